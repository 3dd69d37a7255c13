"""What the operators of a decode step that serves many requests of one model are timed on.

Continuations of a prompt (`KvCache.fork`) hold the same pages for the tokens of the prompt:
`KvCache.find_shared` finds once a step how many, and `KvCache.attend_shared` reads them once for
all in every attention layer.  Requests with low-rank adapters of their own run through one shared
projection, and `AdapterPool.add` adds what each one's adapter gives.  `sample` takes the step's
tokens from its logits: temperature, top-k, top-p and min-p of each request, from random numbers
that are inputs.
"""
import importlib
import math
import random

import torch

own = False

D = 128      # head dimension
TILE = 128   # tokens that are shared or not as a whole
CODE_MAX = 448.0  # largest E4M3 value


def listed():
    return [
        # one request's token: latency
        _sample("sample_1x131072", 1, 131072, "float32", "nucleus", logprobs=True),
        # a decode batch whose requests have parameters of their own, some of them masked by a grammar
        _sample("sample_64x131072", 64, 131072, "float32", "mixed", logprobs=True),
        # a batch with one setting for all, logits as the projection's bf16 rows of a padded vocabulary
        _sample("sample_37x50001", 37, 50001, "bfloat16", "top_k_top_p"),
        # rollouts: a large batch, the distribution as it is
        _sample("sample_256x131072", 256, 131072, "float32", "plain"),
        # eight continuations of a short prompt: latency
        _shared("shared_8x1000", 1, 8, 0, 1000, 60, 1, 32, 8),
        # sixty-four continuations of a long prompt, a token each
        _shared("shared_64x8192", 1, 64, 0, 8192, 200, 1, 32, 8),
        # sixteen continuations of each of eight long contexts, drafted tokens to verify, other requests beside
        _shared("shared_8x16x16384", 8, 16, 5, 16384, 300, 4, 32, 2),
        # what such a step asks once: which tokens are shared
        _find("find_4x8x1000", 4, 8, 0, 1000, 60, 1),
        _find("find_8x16x16384", 8, 16, 5, 16384, 300, 4),
        # one request's token through the queries', keys' and values' projection: latency
        _adapters("adapters_1x1", 1, 1, 2688, 4608, 16, 1),
        # a decode batch, most requests with an adapter of their own, drafted tokens to verify
        _adapters("adapters_64x4", 64, 4, 4096, 2688, 64, 48),
        # the prompts of many requests
        _adapters("adapters_23x356", 23, 356, 2688, 4608, 32, 8),
    ]


def _sample(name, rows, vocab, dtype, mode, logprobs=False):
    return _named(name, kind="sample", rows=rows, vocab=vocab, dtype=dtype, mode=mode,
                  logprobs=logprobs)


def _shared(name, groups, members, lone, prompt, length, rows, heads, kv_heads, page_tokens=64):
    """lone: sequences that share with nobody; prompt: the groups' mean shared prompt; length: what
    the sequences hold beside, a mean; rows: the most new rows a sequence has."""
    return _named(name, kind="shared", groups=groups, members=members, lone=lone, prompt=prompt,
                  length=length, rows=rows, heads=heads, kv_heads=kv_heads, page_tokens=page_tokens)


def _find(name, groups, members, lone, prompt, length, rows, page_tokens=64):
    return _named(name, kind="find", groups=groups, members=members, lone=lone, prompt=prompt,
                  length=length, rows=rows, heads=1, kv_heads=1, page_tokens=page_tokens)


def _adapters(name, sequences, rows, inner, outer, rank, adapters):
    """rows: the sequences' mean; inner, outer: what the projection beside takes and gives."""
    return _named(name, kind="adapters", sequences=sequences, rows=rows, inner=inner, outer=outer,
                  rank=rank, adapters=adapters)


def _named(name, **case):
    if name is not None:
        case["name"] = name
    return case


def _log_int(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


HEADS = [(32, 2), (32, 8), (16, 16), (8, 1), (40, 8), (12, 4)]
WIDTHS = [(2688, 4608), (4096, 2688), (2688, 512), (512, 2688), (1024, 1280), (200, 328), (4096, 4096)]


def draw(rng):
    kind = rng.choice(["sample", "sample", "sample", "shared", "shared", "shared", "find", "adapters",
                       "adapters", "adapters"])
    if kind == "sample":
        vocab = _log_int(rng, 1000, 200000)
        rows = _log_int(rng, 1, min(300, 2 ** 25 // vocab))
        return _sample(None, rows, vocab, rng.choice(["float32", "bfloat16"]),
                       rng.choice(["mixed", "mixed", "nucleus", "top_k_top_p", "plain", "min_p"]),
                       logprobs=rng.random() < 0.5)
    if kind == "adapters":
        inner, outer = rng.choice(WIDTHS)
        sequences = _log_int(rng, 1, 64)
        return _adapters(None, sequences, _log_int(rng, 1, 6000 // sequences), inner, outer,
                         rng.choice([8, 16, 16, 24, 32, 64]), _log_int(rng, 1, 48))
    page_tokens = rng.choice([16, 32, 64, 64, 128])
    groups = rng.randint(4, 8) if kind == "find" else _log_int(rng, 1, 8)
    members = _log_int(rng, 2 if kind == "find" else 1, 96 // groups)
    lone, rows = rng.choice([0, 0, 1, 5]), rng.choice([1, 1, 2, 4])
    heads, kv_heads = rng.choice(HEADS)
    most = min(16384, 2 ** 22 // ((groups * members + lone) * max(kv_heads, heads // 16)),
               2 ** 18 // (groups * kv_heads))
    prompt, length = _log_int(rng, 60, most), _log_int(rng, 8, 300)
    if kind == "find":
        return _find(None, groups, members, lone, _log_int(rng, 1000, 16384), length, rows, page_tokens)
    return _shared(None, groups, members, lone, prompt, length, rows, heads, kv_heads, page_tokens)


def _ragged(case, salt, count, mean, least):
    """Lengths around `mean`, the same for every seed: what a pass costs is the case's."""
    rng = random.Random("%s %s %s %s" % (case["kind"], salt, count, mean))
    if count == 1:
        return [max(least, mean)]
    return [max(least, round(mean * rng.uniform(0.1, 1.9))) for _ in range(count)]


def _prompts(case):
    """Tokens of the groups' prompts, all of them near the mean."""
    rng = random.Random("prompts %s %s" % (case["groups"], case["prompt"]))
    return [round(case["prompt"] * rng.uniform(0.8, 1.2)) if case["groups"] > 1 else case["prompt"]
            for _ in range(case["groups"])]


def _new_rows(case):
    rng = random.Random("rows %s %s" % (case["rows"], case["kind"]))
    if case["kind"] == "adapters":
        return _ragged(case, "rows", case["sequences"], case["rows"], 1)
    return [rng.randint(1, case["rows"]) for _ in range(case["groups"] * case["members"] + case["lone"])]


def _lengths(case):
    """Tokens in the cache, the new rows among them; sequences of a group one behind the other."""
    rows = _new_rows(case)
    beside = _ragged(case, "beside", len(rows), case["length"], 1)
    beside = [max(a, b) for a, b in zip(beside, rows)]
    prompts = [n for n in _prompts(case) for _ in range(case["members"])]
    return [n + b for n, b in zip(prompts + [case["prompt"]] * case["lone"], beside)]


def _pages(tokens, case):
    return -(-tokens // case["page_tokens"])


def _pool(case):
    """Rows of the block table, the pages of a group's prompt in each of its rows, and the pool's size."""
    shared = [n // case["page_tokens"] for n in _prompts(case)]  # full pages: a fork copies a partial one
    lengths, members = _lengths(case), case["members"]
    held = [_pages(n, case) for n in lengths]
    in_groups = case["groups"] * members
    total = sum(shared) + sum(h - (shared[i // members] if i < in_groups else 0)
                              for i, h in enumerate(held)) + 3
    order = list(range(total))
    random.Random("%d %d" % (total, len(held))).shuffle(order)
    prompts, rows, at = [], [], 0
    for s in shared:
        prompts.append(order[at:at + s])
        at += s
    for i, h in enumerate(held):
        prompt = prompts[i // members] if i < in_groups else []
        rows.append(prompt + order[at:at + h - len(prompt)])
        at += h - len(prompt)
    return rows, total


class State:
    pass


def prepare(case, seed):
    s = State()
    s.case = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    if case["kind"] == "sample":
        _prepare_sample(s, g, seed)
    elif case["kind"] == "adapters":
        _prepare_adapters(s, g)
    else:
        _prepare_shared(s, g)
    return s


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _prepare_sample(s, g, seed):
    case = s.case
    rows, vocab = case["rows"], case["vocab"]
    stride = -(-vocab // 64) * 64 if case["dtype"] == "bfloat16" else vocab
    logits = _normal(g, rows, stride) * 2.0
    # some tokens stand out, as after a context that says much about the next one
    likely = torch.randint(0, vocab, (rows, 24), generator=g, device="cuda")
    logits.scatter_add_(1, likely, _normal(g, rows, 24).abs() * 4.0 + 2.0)
    mode = case["mode"]
    s.temperature, s.top_k, s.top_p, s.min_p = {
        "nucleus": (0.7, None, 0.95, None), "top_k_top_p": (0.8, 50, 0.9, None),
        "plain": (1.0, None, None, None), "min_p": (1.1, None, None, 0.05), "mixed": (None,) * 4}[mode]
    if mode == "mixed":
        rng = random.Random(seed)
        s.temperature = _vector([rng.choice([0.0, 0.3, 0.7, 1.0, 1.0, 1.3]) for _ in range(rows)], torch.float32)
        s.top_k = _vector([rng.choice([0, 0, 1, 20, 50, 1000, 5000]) for _ in range(rows)], torch.int32)
        s.top_p = _vector([rng.choice([1.0, 1.0, 0.5, 0.9, 0.95, 0.99]) for _ in range(rows)], torch.float32)
        s.min_p = _vector([rng.choice([0.0, 0.0, 0.02, 0.1]) for _ in range(rows)], torch.float32)
        masked = (torch.rand(rows, 1, generator=g, device="cuda") < 0.25) & \
            (torch.rand(rows, stride, generator=g, device="cuda") < 0.9)
        logits.masked_fill_(masked, -math.inf)
    s.logits = logits.to(getattr(torch, case["dtype"]))[:, :vocab]
    s.uniform = torch.rand(rows, generator=g, device="cuda")
    if own:
        s.sampling = importlib.import_module("nemotron-inference_b200.sampling")


def _vector(values, dtype):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _prepare_adapters(s, g):
    case = s.case
    counts, n = _new_rows(case), case["adapters"]
    rows, inner, outer, rank = sum(counts), case["inner"], case["outer"], case["rank"]
    s.rows, s.counts = rows, counts
    s.x = _normal(g, rows, inner).to(torch.bfloat16)
    s.y = (_normal(g, rows, outer) * 2.0).to(torch.bfloat16)
    s.a = (_normal(g, n, rank, inner) * inner ** -0.5).to(torch.bfloat16)
    s.b = (_normal(g, n, outer, rank) * rank ** -0.5).to(torch.bfloat16)
    s.scales = 0.5 + torch.rand(n, generator=g, device="cuda")
    s.which = _which(case)
    s.ids, s.offsets = _vector(s.which, torch.int32), _offsets(counts)
    if own:
        s.pool = importlib.import_module("nemotron-inference_b200.adapters").AdapterPool(s.a, s.b, s.scales)


def _prepare_shared(s, g):
    case = s.case
    hk, p = case["kv_heads"], case["page_tokens"]
    rows, total = _pool(case)
    layers = 2 if case["kind"] == "shared" else 1
    shape = (layers, total, 2, hk, p, D)
    values = _normal(g, *shape) * 96.0
    values[:, :, 0] += 64.0 * _normal(g, layers, 1, hk, 1, D)  # channels of a key head have means of their own
    s.codes = values.clamp_(-CODE_MAX, CODE_MAX).to(torch.float8_e4m3fn)
    del values
    s.exponents = torch.randint(-8, -5, shape[:4], generator=g, device="cuda", dtype=torch.int8)
    s.width = max(1, max(len(r) for r in rows))
    rows = [r + [0] * (s.width - len(r)) for r in rows]
    if case["kind"] == "find":  # in each group one has parted from the others earlier
        rng = random.Random("%s" % g.initial_seed())
        for i, n in enumerate(_prompts(case)):
            row = rows[i * case["members"] + rng.randrange(case["members"])]
            at = rng.randrange(n // p)
            row[at:n // p] = [(page + 1) % total for page in row[at:n // p]]
    s.table = _vector(rows, torch.int32)
    s.lengths = _vector(_lengths(case), torch.int32)
    used = torch.zeros(total, dtype=torch.int32)
    used.index_add_(0, torch.tensor([page for r in rows for page in r]),
                    torch.ones(sum(len(r) for r in rows), dtype=torch.int32))
    s.references = used.cuda()
    counts = _new_rows(case)
    s.offsets, s.rows, s.most = _offsets(counts), sum(counts), max(counts)
    s.sequences = torch.arange(len(rows), dtype=torch.int32, device="cuda")
    s.groups = _vector([i * case["members"] for i in range(case["groups"] + 1)], torch.int32)
    s.layer = layers - 1
    s.q = (_normal(g, s.rows, case["heads"], D) * 0.8).to(torch.bfloat16)
    if own:
        s.cache = importlib.import_module("nemotron-inference_b200.attention").KvCache(
            s.codes, s.exponents, s.table, s.lengths, s.references)
        if case["kind"] == "shared":  # a step's, kept for all of its layers
            s.shared = s.cache.find_shared(s.sequences, s.offsets, s.groups)


def _offsets(counts):
    at = [0]
    for c in counts:
        at.append(at[-1] + c)
    return _vector(at, torch.int32)


def run(s):
    kind = s.case["kind"]
    if kind == "sample":
        if own:
            return s.sampling.sample(s.logits, s.uniform, temperature=s.temperature, top_k=s.top_k, top_p=s.top_p,
                                     min_p=s.min_p, return_logprobs=s.case["logprobs"])
        return _plain_sample(s)
    if kind == "shared":
        if own:
            return s.cache.attend_shared(s.layer, s.q, s.sequences, s.offsets, s.groups, s.shared)
        return _plain_shared(s)
    if kind == "find":
        return s.cache.find_shared(s.sequences, s.offsets, s.groups) if own else _plain_find(s)
    return s.pool.add(s.x, s.y, s.ids, s.offsets) if own else _plain_adapters(s)


def _column(value, default, rows):
    """A parameter for each row, of one for all or none."""
    if isinstance(value, torch.Tensor):
        return value.double()[:, None]
    return torch.full((rows, 1), float(default if value is None else torch.tensor(value, dtype=torch.float32)),
                      dtype=torch.float64, device="cuda")


def _plain_sample(s):
    """Tokens in falling order of their logits, ties by rising number; the first top_k of them; of these as
    many as reach top_p of their sum; of these those of min_p times the largest.  What is left, in rising
    order of the tokens, is shared out from 0 to 1, and the random number falls on one."""
    x = s.logits.double()
    rows, vocab = x.shape
    temperature, top_k = _column(s.temperature, 1.0, rows), _column(s.top_k, 0, rows)
    top_p, min_p = _column(s.top_p, 1.0, rows), _column(s.min_p, 0.0, rows)
    down, order = x.sort(dim=1, descending=True, stable=True)
    rank = torch.arange(vocab, device="cuda")
    greedy = ~(temperature > 0)
    weights = ((down - down[:, :1]) / torch.where(greedy, 1.0, temperature)).exp()
    weights = torch.where((top_k >= 1) & (rank >= top_k), 0.0, weights)
    upto = weights.cumsum(dim=1)
    before = torch.cat([torch.zeros_like(upto[:, :1]), upto[:, :-1]], dim=1)
    kept = ((top_p >= 1) | (before < top_p * upto[:, -1:])) & (weights >= min_p.clamp(max=1.0)) & (weights > 0) & ~greedy
    kept |= rank == 0
    in_order = torch.zeros_like(weights).scatter_(1, order, torch.where(kept, weights, 0.0))
    upto = in_order.cumsum(dim=1)
    token = (upto <= s.uniform.double()[:, None] * upto[:, -1:]).sum(dim=1, keepdim=True)
    if not s.case["logprobs"]:
        return token[:, 0].int()
    logprob = x.gather(1, token) - down[:, :1] - (down - down[:, :1]).exp().sum(dim=1, keepdim=True).log()
    return token[:, 0].int(), logprob[:, 0].float()


def _plain_shared(s):
    """New row j of a sequence stands at position length - rows + j and sees every token up to it."""
    hk, p = s.case["kv_heads"], s.case["page_tokens"]
    which = s.sequences.long()
    pages = s.table[which].long()
    values = s.codes[s.layer][pages].float()  # [n, width, 2, hk, p, D]
    values *= torch.exp2(s.exponents[s.layer][pages].float())[..., None, None]
    kv = values.permute(2, 0, 3, 1, 4, 5).flatten(3, 4)  # [2, n, hk, tokens, D]
    counts = (s.offsets[1:] - s.offsets[:-1]).long()
    j = torch.arange(s.most, device="cuda")
    row = (s.offsets[:-1, None].long() + j).clamp(max=s.rows - 1)
    q = s.q.float()[row].unflatten(2, (hk, -1)).transpose(1, 2)  # [n, hk, most, group, D]
    scores = (q.flatten(2, 3) @ kv[0].transpose(2, 3)) * D ** -0.5
    position = s.lengths[which].long()[:, None] - counts[:, None] + j
    seen = torch.arange(s.width * p, device="cuda") <= position[..., None]  # [n, most, tokens]
    scores = scores.unflatten(2, (s.most, -1)).masked_fill(~seen[:, None, :, None], -math.inf)
    weights = (scores - scores.amax(dim=4, keepdim=True)).exp()
    out = (weights.flatten(2, 3) @ kv[1]) / weights.sum(dim=4).flatten(2, 3)[..., None]
    out = out.unflatten(2, (s.most, -1)).transpose(1, 2).flatten(2, 3)  # [n, most, heads, D]
    return out[j[None, :] < counts[:, None]].to(torch.bfloat16)


def _plain_find(s):
    """Whole tiles of tokens, before every new row, whose pages all members of a group with new rows have in
    common, if two or more have some."""
    p, n = s.case["page_tokens"], s.sequences.numel()
    which = s.sequences.long()
    entry = torch.arange(n, device="cuda")
    group = torch.searchsorted(s.groups, entry.int(), right=True) - 1
    inside = (group >= 0) & (group < s.groups.numel() - 1)
    group = torch.where(inside, group, 0)
    counts = (s.offsets[1:] - s.offsets[:-1]).long()
    active = inside & (counts > 0)
    first = torch.full((s.groups.numel() - 1,), n, device="cuda")
    first.index_reduce_(0, group, torch.where(active, entry, n), "amin")
    first = first.clamp(max=n - 1)[group]
    pages = s.table[which]
    same = (pages == pages[first]).long().cumprod(dim=1).sum(dim=1) * p
    most = torch.minimum(same, s.lengths[which].long() - counts)
    no_limit = torch.iinfo(torch.int32).max
    common = torch.full((s.groups.numel() - 1,), no_limit, device="cuda")
    common.index_reduce_(0, group, torch.where(active, most, no_limit), "amin")
    members = torch.zeros_like(common).index_add_(0, group, active.long())
    tokens = torch.where(members >= 2, common // TILE * TILE, 0)
    return torch.where(inside, tokens[group], 0).int()


def _plain_adapters(s):
    """All adapters' products, of which each row keeps its own's."""
    n, rank = s.a.shape[:2]
    row = torch.arange(s.rows, device="cuda")
    mine = s.ids.long()[torch.searchsorted(s.offsets, row.int(), right=True) - 1]
    inside = (s.x.float() @ s.a.float().flatten(0, 1).T).unflatten(1, (n, rank))
    keep = (mine[:, None] == torch.arange(n, device="cuda")) * s.scales
    inside = (inside * keep[:, :, None]).flatten(1, 2)
    return (s.y.float() + inside @ s.b.float().transpose(1, 2).flatten(0, 1)).to(torch.bfloat16)


def work(case):
    kind = case["kind"]
    if kind == "sample":
        elements = case["rows"] * case["vocab"]
        size = 2 if case["dtype"] == "bfloat16" else 4
        return {"bytes": size * elements + 12 * case["rows"], "flops": elements}
    counts = _new_rows(case)
    if kind == "adapters":
        which = _which(case)
        active = sum(c for c, a in zip(counts, which) if a >= 0)
        used = len({a for a in which if a >= 0})
        inner, outer, rank = case["inner"], case["outer"], case["rank"]
        return {"bytes": 2 * active * inner + 4 * sum(counts) * outer + 2 * used * rank * (inner + outer),
                "flops": 2 * active * rank * (inner + outer)}
    lengths, hk, hq = _lengths(case), case["kv_heads"], case["heads"]
    p, members = case["page_tokens"], case["members"]
    prompts = [n // p * p for n in _prompts(case)]
    if kind == "find":
        pages = sum(n // p for n in prompts) * members
        return {"bytes": 4 * pages + 16 * len(counts), "flops": 0}
    alone = sum(n - (prompts[i // members] if i < case["groups"] * members else 0) for i, n in enumerate(lengths))
    tokens = sum(prompts) + alone
    pairs = sum(c * n - c * (c - 1) // 2 for n, c in zip(lengths, counts))
    return {"bytes": 2 * hk * (D * tokens + tokens // p) + 4 * D * hq * sum(counts), "flops": 4 * D * hq * pairs}


def _which(case):
    """The sequences' adapters; one request in eight has none."""
    counts, n = _new_rows(case), case["adapters"]
    rng = random.Random("adapters %d %d" % (len(counts), n))
    return [-1 if len(counts) > 1 and rng.random() < 0.125 else rng.randrange(n) for _ in counts]


def exact(case, seed):
    """The operators from their definitions, in 64 bits."""
    s = prepare(case, seed)
    if case["kind"] == "sample":
        return _exact_sample(s)
    if case["kind"] == "adapters":
        return _exact_adapters(s)
    if case["kind"] == "shared":
        return _exact_shared(s)
    return None  # whole numbers that nothing is computed for


def _of_row(value, default, i):
    if isinstance(value, torch.Tensor):
        return float(value[i])
    return default if value is None else float(torch.tensor(value, dtype=torch.float32))


def _exact_sample(s):
    tokens, logprobs = [], []
    for i in range(s.case["rows"]):
        x = s.logits[i].double()
        temperature, top_k = _of_row(s.temperature, 1.0, i), _of_row(s.top_k, 0, i)
        top_p, min_p = _of_row(s.top_p, 1.0, i), _of_row(s.min_p, 0.0, i)
        if temperature <= 0:
            token = int((x == x.max()).nonzero()[0])
        else:
            order = x.neg().sort(stable=True).indices
            probabilities = torch.softmax(x / temperature, dim=0)[order]
            if top_k >= 1:
                order, probabilities = order[:int(top_k)], probabilities[:int(top_k)]
            if top_p < 1:
                reached = probabilities.cumsum(0) >= top_p * probabilities.sum()
                count = int(reached.nonzero()[0]) + 1 if bool(reached.any()) else order.numel()
                order, probabilities = order[:count], probabilities[:count]
            some = probabilities >= min_p * probabilities[0]
            order, probabilities = order[some], probabilities[some]
            rising = order.argsort()
            order, upto = order[rising], probabilities[rising].cumsum(0)
            at = int(torch.searchsorted(upto, s.uniform[i].double() * upto[-1], right=True))
            token = int(order[min(at, order.numel() - 1)])
        tokens.append(token)
        logprobs.append(float(torch.log_softmax(x, dim=0)[token]))
    tokens = _vector(tokens, torch.int32)
    return (tokens, _vector(logprobs, torch.float64)) if s.case["logprobs"] else tokens


def _exact_adapters(s):
    out, start = s.y.double(), 0
    for c, which in zip(s.counts, s.which):
        if which >= 0:
            inside = s.x[start:start + c].double() @ s.a[which].double().T
            out[start:start + c] += float(s.scales[which]) * (inside @ s.b[which].double().T)
        start += c
    return out


def _exact_shared(s):
    hq, hk = s.case["heads"], s.case["kv_heads"]
    out = torch.zeros((s.rows, hq, D), dtype=torch.float64, device="cuda")
    start = 0
    for i, (n, c) in enumerate(zip(_lengths(s.case), _new_rows(s.case))):
        pages = s.table[i, :_pages(n, s.case)].long()
        scale = torch.pow(2.0, s.exponents[s.layer, pages].double())[..., None, None]
        values = (s.codes[s.layer, pages].double() * scale).permute(1, 2, 0, 3, 4).flatten(2, 3)[:, :, :n]
        at = torch.arange(n, device="cuda")
        seen = at[None, :] <= (n - c + torch.arange(c, device="cuda"))[:, None]
        q = s.q[start:start + c].double().unflatten(1, (hk, hq // hk)).permute(1, 2, 0, 3)  # [hk, group, c, D]
        scores = q @ values[0][:, None].transpose(2, 3) / math.sqrt(D)
        weights = torch.softmax(scores.masked_fill(~seen, -math.inf), dim=3)
        out[start:start + c] = (weights @ values[1][:, None]).permute(2, 0, 1, 3).flatten(1, 2)
        start += c
    return out
