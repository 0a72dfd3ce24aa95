"""Three operators of serving several answers to one prompt, as cases that can be timed and compared: the draw of the next
id behind filters (top-k, top-p, min-p), attention of decoding rows whose caches begin with the same pages, and the copies
of cache pages that a fork of a request makes.  `run` gives each in its plain form (elementary torch operations) or, with
`own`, through the framework's entry point.

Sizes are those of the benchmark's configurations, or generic.
"""
import math

import torch

own = False

DEVICE = "cuda:0"
F32, F64 = torch.float32, torch.float64
TYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}
# query heads, key/value heads, lanes a head
HEADS = {"14/2x64": (14, 2, 64), "12/2x128": (12, 2, 128), "28/4x128": (28, 4, 128), "8/8x64": (8, 8, 64), "16/1x128": (16, 1, 128)}
NONE = -1


def listed():
    return [
        # the next id of one chat, as a model card's settings ask for it: latency alone
        {"name": "sample_1", "kind": "sample", "rows": 1, "vocab": 151936, "spread": 2.0, "settings": "all"},
        # eight answers drawn from the nucleus of a confident model
        {"name": "sample_8", "kind": "sample", "rows": 8, "vocab": 151936, "spread": 2.0, "settings": "nucleus"},
        # a full batch in which every request has settings of its own, greedy ones and unfiltered ones among them
        {"name": "sample_64_mixed", "kind": "sample", "rows": 64, "vocab": 152064, "spread": 1.5, "settings": "mixed"},
        # an odd vocabulary and nearly flat logits: large candidate sets
        {"name": "sample_37_flat", "kind": "sample", "rows": 37, "vocab": 49999, "spread": 0.7, "settings": "warm"},
        # four answers behind a short prompt
        {"name": "shared_4_short", "kind": "shared", "heads": "14/2x64", "dtype": "bfloat16", "page": 16, "rows": 4, "sets": 1, "alone": 0,
         "prefix": 512, "own": 64, "sink": False, "softcap": 0.0},
        # sixteen answers behind a document
        {"name": "shared_16", "kind": "shared", "heads": "12/2x128", "dtype": "bfloat16", "page": 16, "rows": 16, "sets": 1, "alone": 0,
         "prefix": 4096, "own": 512, "sink": False, "softcap": 0.0},
        # a full batch of answers to one long prompt
        {"name": "shared_64_long", "kind": "shared", "heads": "28/4x128", "dtype": "bfloat16", "page": 16, "rows": 64, "sets": 1, "alone": 0,
         "prefix": 8192, "own": 1024, "sink": False, "softcap": 0.0},
        # three uneven sets beside requests that share nothing, with a softmax sink and capped scores
        {"name": "shared_33_sets", "kind": "shared", "heads": "14/2x64", "dtype": "bfloat16", "page": 8, "rows": 33, "sets": 3, "alone": 5,
         "prefix": 2048, "own": 333, "sink": True, "softcap": 30.0},
        # the true 32-bit path, as results are checked with it
        {"name": "shared_8_f32", "kind": "shared", "heads": "14/2x64", "dtype": "float32", "page": 16, "rows": 8, "sets": 1, "alone": 0,
         "prefix": 1024, "own": 200, "sink": False, "softcap": 0.0},
        # three more answers to a prompt that ends inside a page
        {"name": "fork_3", "kind": "copy", "planes": 48, "heads": "14/2x64", "dtype": "bfloat16", "page": 16, "pairs": 3, "sources": 1},
        # a batch's worth of answers of a large model
        {"name": "fork_63", "kind": "copy", "planes": 56, "heads": "28/4x128", "dtype": "bfloat16", "page": 16, "pairs": 63, "sources": 1},
        # seven prompts forked at once, 32-bit, pages of an odd size
        {"name": "fork_21_f32", "kind": "copy", "planes": 30, "heads": "12/2x128", "dtype": "float32", "page": 21, "pairs": 21, "sources": 7},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["sample", "shared", "shared", "copy"])
    if kind == "sample":
        return {"kind": kind, "rows": _log(rng, 1, 64), "vocab": _log(rng, 300, 152064), "spread": round(rng.uniform(0.5, 3.0), 2),
                "settings": rng.choice(["all", "nucleus", "mixed", "warm"])}
    if kind == "copy":
        pairs = _log(rng, 1, 63)
        return {"kind": kind, "planes": 2 * _log(rng, 1, 28), "heads": rng.choice(sorted(HEADS)), "dtype": rng.choice(sorted(TYPES)),
                "page": _log(rng, 5, 24), "pairs": pairs if pairs < 24 else pairs // 2, "sources": rng.randint(1, 3)}
    dtype = rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"])
    small = dtype == "float32"
    rows = _log(rng, 2, 16 if small else 64)
    return {"kind": kind, "heads": rng.choice(["14/2x64", "12/2x128", "8/8x64"] if small else sorted(HEADS)), "dtype": dtype,
            "page": rng.choice([8, 16, 16, 32]), "rows": rows, "sets": rng.randint(1, max(1, min(4, rows // 2))), "alone": rng.randint(0, rows // 4),
            "prefix": _log(rng, 64, 2000 if small else 8000), "own": _log(rng, 1, 500), "sink": rng.random() < 0.3,
            "softcap": rng.choice([0.0, 0.0, 30.0])}


# ---- inputs --------------------------------------------------------------------------------------------------------
def _settings(kind, rows, host):
    """Temperature, top-k (0: off), top-p (1: off) and min-p (0: off) of each row."""
    spread = torch.rand(4, rows, generator=host)
    if kind == "all":
        return torch.full((rows,), 0.7), torch.full((rows,), 20, dtype=torch.int32), torch.full((rows,), 0.8), torch.full((rows,), 0.01)
    if kind == "nucleus":
        return 0.6 + 0.4 * spread[0], torch.zeros(rows, dtype=torch.int32), 0.85 + 0.1 * spread[1], torch.zeros(rows)
    if kind == "warm":
        return 1.0 + 0.5 * spread[0], torch.zeros(rows, dtype=torch.int32), 0.9 + 0.1 * spread[1], 0.05 * spread[2] * (spread[3] < 0.5)
    turn = torch.arange(rows) % 6
    temperature = torch.where(turn == 0, torch.zeros(rows), 0.3 + 1.2 * spread[0])
    top_k = torch.where((turn == 1) | (turn == 4), (1 + 200 * spread[1]).to(torch.int32), torch.zeros(rows, dtype=torch.int32))
    top_p = torch.where((turn == 2) | (turn == 4), 0.5 + 0.5 * spread[2], torch.ones(rows))
    min_p = torch.where((turn == 3) | (turn == 4), 0.1 * spread[3], torch.zeros(rows))
    return temperature, top_k, top_p, min_p


def _prepare_sample(case, seed, host, device):
    rows, vocab = case["rows"], case["vocab"]
    logits = case["spread"] * torch.randn(rows, vocab, generator=device, device=DEVICE)
    # the ids that the model means, some nats above the others; one in each fortieth of the vocabulary
    part = vocab // 40
    meant = (torch.arange(40) * part + torch.randint(0, part, (rows, 40), generator=host)).to(DEVICE)
    lift = (3.0 * torch.empty(rows, 40).exponential_(generator=host)).to(DEVICE)
    logits.scatter_add_(1, meant, lift)
    temperature, top_k, top_p, min_p = (t.to(DEVICE) for t in _settings(case["settings"], rows, host))
    uniform = (torch.randint(0, 1 << 24, (rows,), generator=host).to(F32) / (1 << 24)).to(DEVICE)
    return {"logits": logits, "temperature": temperature, "top_k": top_k, "top_p": top_p, "min_p": min_p, "uniform": uniform,
            "out": torch.zeros(rows, dtype=torch.int32, device=DEVICE)}


def _lengths(case, host):
    """Per row: its set (NONE: alone), the keys it shares with the set, its keys in all."""
    rows, page = case["rows"], case["page"]
    together = rows - case["alone"]
    sets, per_set = [], []
    for s in range(case["sets"]):
        least = case["prefix"] if s == 0 else case["prefix"] // 3
        per_set.append(max(1, int(torch.randint(least, case["prefix"] + 1, (1,), generator=host)) // page) * page)
    weights = [1.0 + 0.7 * s for s in range(case["sets"])]
    ends = [round(together * sum(weights[:s + 1]) / sum(weights)) for s in range(case["sets"])]
    for r in range(rows):
        sets.append(next(s for s, end in enumerate(ends) if r < end) if r < together else NONE)
    shared = [per_set[s] if s != NONE else 0 for s in sets]
    own_keys = torch.randint(max(1, case["own"] // 4), case["own"] + 1, (rows,), generator=host).tolist()
    return sets, shared, [a + b for a, b in zip(shared, own_keys)]


def _prepare_shared(case, seed, host, device):
    nh, nkv, d = HEADS[case["heads"]]
    dtype, page, rows = TYPES[case["dtype"]], case["page"], case["rows"]
    sets, shared, total = _lengths(case, host)
    blocks = [-(-n // page) for n in total]
    heads_of_sets = {s: shared[sets.index(s)] // page for s in set(sets) if s != NONE}
    n_pages = sum(heads_of_sets.values()) + sum(b - k // page for b, k in zip(blocks, shared))
    free = iter(torch.randperm(n_pages, generator=host).tolist())
    begins = {s: [next(free) for _ in range(n)] for s, n in sorted(heads_of_sets.items())}
    table = torch.full((rows, max(blocks)), NONE, dtype=torch.int32)
    for r in range(rows):
        pages = list(begins.get(sets[r], []))
        pages += [next(free) for _ in range(blocks[r] - len(pages))]
        table[r, :len(pages)] = torch.tensor(pages, dtype=torch.int32)
    # the rows of a step come in any order
    order = torch.randperm(rows, generator=host).tolist()
    table, shared, total, sets = table[order], [shared[i] for i in order], [total[i] for i in order], [sets[i] for i in order]
    # the plan that goes with the batch: rows set by set, cut into tiles of as many rows as two tiles of 128 heads hold
    most = 2 * (128 // (nh // nkv))
    members, tiles = [], []
    for s in sorted(begins):
        of_set = [r for r in range(rows) if sets[r] == s]
        for at in range(0, len(of_set), most):
            part = of_set[at:at + most]
            tiles.append([len(members), len(part), shared[part[0]], 0])
            members += part
    pool = lambda: torch.randn(n_pages * page, nkv, d, generator=device, device=DEVICE).to(dtype)  # noqa: E731
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEVICE)  # noqa: E731
    return {"case": case, "q": (1.3 * torch.randn(rows, nh * d, generator=device, device=DEVICE)).to(dtype), "k": pool(), "v": pool(),
            "out": torch.zeros(rows, nh * d, dtype=dtype, device=DEVICE), "table": table.to(DEVICE), "row_req": ints(list(range(rows))),
            "pos": ints([n - 1 for n in total]), "shared": ints(shared), "members": ints(members), "tiles": ints(tiles).view(-1, 4),
            "sink": torch.randn(nh, generator=device, device=DEVICE) if case["sink"] else None, "longest": max(total)}


def _copies(case, host):
    """(pages of the pool, [(source page, destination page, rows)]): the last pages of some prompts, each copied for the forks of its own."""
    pages = 2 * (case["pairs"] + case["sources"])
    free = torch.randperm(pages, generator=host).tolist()
    sources = [(free.pop(), int(torch.randint(1, case["page"], (1,), generator=host))) for _ in range(case["sources"])]
    return pages, [(sources[i % len(sources)][0], free.pop(), sources[i % len(sources)][1]) for i in range(case["pairs"])]


def _prepare_copy(case, seed, host, device):
    _, nkv, d = HEADS[case["heads"]]
    pages, pairs = _copies(case, host)
    pool = torch.randn(case["planes"] // 2, 2, pages * case["page"], nkv, d, generator=device, device=DEVICE).to(TYPES[case["dtype"]])
    return {"case": case, "pool": pool, "pairs": pairs}


def prepare(case, seed):
    host, device = torch.Generator().manual_seed(seed), torch.Generator(DEVICE).manual_seed(seed)
    make = {"sample": _prepare_sample, "shared": _prepare_shared, "copy": _prepare_copy}[case["kind"]]
    return {"kind": case["kind"], **make(case, seed, host, device)}


# ---- the plain forms -----------------------------------------------------------------------------------------------
def _plain_sample(s):
    # sums and shares in 64 bits: a draw lies as near to its neighbour as the smallest weight
    values, ids = torch.sort(s["logits"], dim=1, descending=True, stable=True)          # equal logits: the lower id first
    t = s["temperature"].to(F64)[:, None]
    weights = torch.exp((values.to(F64) - values[:, :1].to(F64)) / torch.where(t > 0, t, torch.ones_like(t)))
    place = torch.arange(values.shape[1], device=values.device)[None, :]
    k = s["top_k"][:, None]
    weights = torch.where((k <= 0) | (place < k), weights, torch.zeros_like(weights))
    sums = torch.cumsum(weights, dim=1)
    p = s["top_p"].to(F64)[:, None]
    kept = (place == 0) | (p >= 1) | (sums - weights < p * sums[:, -1:])
    kept &= (weights >= s["min_p"].to(F64)[:, None]) & (weights > 0)
    share = torch.where(kept, sums, torch.zeros_like(sums)).amax(dim=1, keepdim=True)
    at = (sums <= s["uniform"].to(F64)[:, None] * share).sum(dim=1, keepdim=True)
    at = torch.where(t > 0, torch.minimum(at, kept.sum(dim=1, keepdim=True) - 1), torch.zeros_like(at))
    return torch.gather(ids, 1, at)[:, 0].to(torch.int32)


def _plain_shared(s):
    nh, nkv, d = HEADS[s["case"]["heads"]]
    page, rows, n = s["case"]["page"], s["q"].shape[0], s["longest"]
    key = torch.arange(n, device=DEVICE)
    slots = s["table"][s["row_req"].long()][:, key // page].clamp_min(0).long() * page + key % page          # [rows, n]
    q = s["q"].to(F32).view(rows, nkv, nh // nkv, d)
    k, v = s["k"][slots].to(F32), s["v"][slots].to(F32)                                                       # [rows, n, nkv, d]
    scores = torch.matmul(q, k.permute(0, 2, 3, 1)) * (1.0 / math.sqrt(d))                                    # [rows, nkv, group, n]
    cap = s["case"]["softcap"]
    if cap:
        scores = cap * torch.tanh(scores / cap)
    hidden = key[None, :] > s["pos"][:, None]
    scores = torch.where(hidden[:, None, None, :], torch.full_like(scores, -math.inf), scores)
    top = scores.amax(dim=-1, keepdim=True)
    if s["sink"] is not None:
        sink = s["sink"].view(1, nkv, nh // nkv, 1)
        top = torch.maximum(top, sink)
    p = torch.exp(scores - top)
    total = p.sum(dim=-1, keepdim=True)
    if s["sink"] is not None:
        total = total + torch.exp(sink - top)
    return (torch.matmul(p, v.permute(0, 2, 1, 3)) / total).reshape(rows, nh * d).to(s["q"].dtype)


def _plain_copy(s):
    page, pool = s["case"]["page"], s["pool"]
    pairs = torch.tensor(s["pairs"], device=DEVICE)
    offset = torch.arange(page, device=DEVICE)[None, :]
    wanted = offset < pairs[:, 2:3]
    source, target = (pairs[:, 0:1] * page + offset)[wanted], (pairs[:, 1:2] * page + offset)[wanted]
    pool[:, :, target] = pool[:, :, source]
    return pool


def run(state):
    if own:
        from tokenizer_b200.kernels import ops
    if state["kind"] == "sample":
        if own:
            ops.sample_filtered(state["logits"], state["temperature"], state["top_k"], state["top_p"], state["min_p"], state["uniform"], state["out"])
            return state["out"]
        return _plain_sample(state)
    case = state["case"]
    if state["kind"] == "copy":
        if own:
            ops.copy_pages(state["pool"], case["page"], state["pairs"])
            return state["pool"]
        return _plain_copy(state)
    if own:
        nh, nkv, d = HEADS[case["heads"]]
        ops.shared_prefix_attention(state["q"], state["k"], state["v"], state["out"], state["table"], state["row_req"], state["pos"],
                                    state["shared"], state["members"], state["tiles"], nh, nkv, d, case["page"], 1.0 / math.sqrt(d),
                                    sink=state["sink"], softcap=case["softcap"] or None)
        return state["out"]
    return _plain_shared(state)


# ---- what a pass cannot do without ---------------------------------------------------------------------------------
def work(case):
    if case["kind"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": 4 * n, "flops": 4 * n}
    nh, nkv, d = HEADS[case["heads"]]
    size = 2 if case["dtype"] == "bfloat16" else 4
    if case["kind"] == "copy":
        rows = case["planes"] * nkv * d * size * (case["page"] / 2)             # half a page on the average
        return {"bytes": rows * (case["pairs"] + case["sources"]), "flops": 0}
    own_keys = case["rows"] * (case["own"] + case["own"] // 4) / 2
    prefix = case["prefix"] * (1 + (case["sets"] - 1) * 2 / 3)
    together = (case["rows"] - case["alone"]) * case["prefix"] * (1 if case["sets"] == 1 else 0.75)
    return {"bytes": 2 * (prefix + own_keys) * nkv * d * size + 2 * case["rows"] * nh * d * size,
            "flops": 4 * nh * d * (together + own_keys)}


# ---- the definitions, in 64 bits -----------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "sample":
        return None                       # ids are whole numbers
    if case["kind"] == "copy":
        page, pool = case["page"], s["pool"]
        for source, target, rows in s["pairs"]:
            pool[:, :, target * page:target * page + rows] = pool[:, :, source * page:source * page + rows].clone()
        return pool.to(F64)
    nh, nkv, d = HEADS[case["heads"]]
    rows, page = case["rows"], case["page"]
    answer = torch.empty(rows, nh, d, dtype=F64, device=DEVICE)
    for r, n in enumerate((s["pos"] + 1).tolist()):
        pages = s["table"][r, :-(-n // page)].long()
        k, v = (s[name].view(-1, page, nkv, d)[pages].reshape(-1, nkv, d)[:n].to(F64) for name in "kv")
        for h in range(nh):
            x = (k[:, h * nkv // nh] @ s["q"][r, h * d:(h + 1) * d].to(F64)) / math.sqrt(d)
            if case["softcap"]:
                x = case["softcap"] * torch.tanh(x / case["softcap"])
            extra = s["sink"][h:h + 1].to(F64) if case["sink"] else x[:0]
            share = torch.softmax(torch.cat([x, extra]), dim=0)[:n]
            answer[r, h] = share @ v[:, h * nkv // nh]
    return answer.view(rows, nh * d)
