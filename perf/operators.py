"""What the attention operators are timed on: prompts, the paged 8-bit cache, and its pages.

A serving loop runs a prompt through `attention_prefill` and writes its keys and values into a
`KvCache` (`append`); a decode step appends a row or a few drafted rows per sequence and attends
over the cache (`attend`); sampling several continuations of one prompt forks its pages (`fork`);
a pool with holes is made dense again (`compact`).

The cache is one tensor of E4M3 codes [layers, pages, 2 (keys, values), kv_heads, page_tokens, 128]
and one of exponents [layers, pages, 2, kv_heads]: a code stands for its value times 2^exponent.
The plain forms below state the operators in elementary torch operations on the same tensors.
"""
import importlib
import math
import random

import torch

own = False

D = 128  # head dimension
CODE_MAX = 448.0  # largest E4M3 value
EXPONENT_MIN, EXPONENT_MAX = -32, 32


def listed():
    return [
        # a short prompt of one request: launches and latency
        _prefill("prefill_17", 17, 1, 32, 2),
        # seven requests of odd lengths batched together; the row sums' logarithms are kept
        _prefill("prefill_packed_1000", 1000, 7, 32, 8, lse=True),
        # a prefill chunk of many requests
        _prefill("prefill_packed_8190", 8190, 23, 32, 8),
        # one long prompt
        _prefill("prefill_8192", 8192, 1, 32, 2),
        # one sequence being decoded: latency
        _attend("attend_1x1500", 1, 1500, 1, 32, 2),
        # a full decode batch of ragged lengths, a token each
        _attend("attend_64x2048", 64, 2048, 1, 32, 8),
        # one sequence at the 64k context
        _attend("attend_1x65536", 1, 65536, 1, 32, 8),
        # a batch whose sequences each verify up to eight drafted tokens, sixteen heads to a key head
        _attend("attend_drafts_48x8192", 48, 8192, 8, 32, 2),
        # the new rows of a decode batch: latency
        _append("append_64x1", 64, 1, 700, 2),
        # the rows of a prefill chunk, into pages that some sequences have begun
        _append("append_8190", 23, 356, 100, 8),
        # eight continuations of each of sixteen prompts: shared pages, copies of the last ones
        _fork("fork_16x8", 16, 8, 900, 8, 8),
        # a pool with holes between its pages, as finished requests leave it
        _compact("compact_96", 96, 1000, 8, 4, 0.5),
    ]


def _prefill(name, tokens, sequences, heads, kv_heads, lse=False):
    return _named(name, kind="prefill", tokens=tokens, sequences=sequences, heads=heads,
                  kv_heads=kv_heads, lse=lse)


def _attend(name, sequences, length, rows, heads, kv_heads, page_tokens=64):
    """length: the sequences' mean; rows: the most new rows a sequence has."""
    return _named(name, kind="attend", sequences=sequences, length=length, rows=rows, heads=heads,
                  kv_heads=kv_heads, page_tokens=page_tokens)


def _append(name, sequences, rows, length, kv_heads, page_tokens=64):
    """rows, length: the means of the new rows and of what the sequences held before."""
    return _named(name, kind="append", sequences=sequences, rows=rows, length=length,
                  kv_heads=kv_heads, page_tokens=page_tokens)


def _fork(name, prompts, samples, length, layers, kv_heads, page_tokens=64):
    return _named(name, kind="fork", sequences=prompts, samples=samples, length=length,
                  layers=layers, kv_heads=kv_heads, page_tokens=page_tokens)


def _compact(name, sequences, length, layers, kv_heads, share, page_tokens=64):
    """share: of the pool's pages that are in use."""
    return _named(name, kind="compact", sequences=sequences, length=length, layers=layers,
                  kv_heads=kv_heads, share=share, page_tokens=page_tokens)


def _named(name, **case):
    if name is not None:
        case["name"] = name
    return case


def _log_int(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


HEADS = [(32, 2), (32, 8), (16, 16), (8, 1), (24, 8), (40, 8), (12, 4)]


def draw(rng):
    kind = rng.choice(["prefill", "prefill", "attend", "attend", "attend", "append", "fork", "compact"])
    page_tokens = rng.choice([16, 32, 64, 64, 128])
    heads, kv_heads = rng.choice(HEADS)
    if kind == "prefill":
        most = int(8192 * math.sqrt(min(1.0, 32 / heads)))
        tokens = _log_int(rng, 1, most)
        return _prefill(None, tokens, min(tokens, _log_int(rng, 1, 40)), heads, kv_heads,
                        lse=rng.random() < 0.5)
    if kind == "attend":
        sequences = _log_int(rng, 1, 128)
        length = _log_int(rng, 1, min(65536, 2 ** 19 // (sequences * kv_heads)))
        return _attend(None, sequences, length, rng.choice([1, 1, 2, 3, 4, 5, 8]), heads, kv_heads,
                       page_tokens)
    if kind == "append":
        sequences = _log_int(rng, 1, 64)
        return _append(None, sequences, _log_int(rng, 1, 8190 // sequences), _log_int(rng, 1, 1000),
                       rng.choice([1, 2, 4, 8]), page_tokens)
    layers, kv_heads = rng.choice([1, 3, 8]), rng.choice([1, 2, 4, 8])
    if kind == "fork":
        return _fork(None, _log_int(rng, 1, 16), _log_int(rng, 1, 8), _log_int(rng, 1, 900), layers,
                     kv_heads, page_tokens)
    return _compact(None, _log_int(rng, 1, 96), _log_int(rng, 1, 1000), layers, min(kv_heads, 4),
                    rng.uniform(0.2, 0.9), page_tokens)


def _ragged(case, salt, mean, least, most=None):
    """Lengths around `mean`, the same for every seed: what a pass costs is the case's."""
    rng = random.Random("%s %s %s %s" % (case["kind"], salt, case["sequences"], mean))
    n = case["sequences"]
    if n == 1:
        got = [mean]
    else:
        got = [round(mean * rng.uniform(0.1, 1.9)) for _ in range(n)]
    return [min(max(least, g), most or max(least, g)) for g in got]


def _prompt_lengths(case):
    """Sequences of a packed batch: they add up to its tokens; one in eight is empty."""
    rng = random.Random("%d %d" % (case["tokens"], case["sequences"]))
    n = case["sequences"]
    weights = [0.0 if n > 1 and rng.random() < 0.125 else rng.uniform(0.1, 1.9) for _ in range(n)]
    weights[rng.randrange(n)] += 0.5
    whole = [int(case["tokens"] * w / sum(weights)) for w in weights]
    whole[max(range(n), key=lambda i: whole[i])] += case["tokens"] - sum(whole)
    return whole


def _new_rows(case):
    if case["kind"] == "attend":
        rng = random.Random("rows %d %d" % (case["rows"], case["sequences"]))
        return [case["rows"] if case["sequences"] == 1 else rng.randint(1, case["rows"])
                for _ in range(case["sequences"])]
    return _ragged(case, "rows", case["rows"], 1)


def _lengths(case):
    """Tokens in the cache, the new rows among them."""
    if case["kind"] == "append":
        return [h + r for h, r in zip(_ragged(case, "held", case["length"], 0), _new_rows(case))]
    lengths = _ragged(case, "length", case["length"], 1)
    if case["kind"] == "attend":
        lengths = [max(a, r) for a, r in zip(lengths, _new_rows(case))]
    return lengths


def _pages(tokens, case):
    return -(-tokens // case["page_tokens"])


def _last_is_partial(tokens, case):
    return tokens % case["page_tokens"] != 0


def _page_bytes(case):
    """One page of all layers: codes and exponents."""
    return case.get("layers", 1) * 2 * case["kv_heads"] * (case["page_tokens"] * D + 1)


def _pool(case):
    """Rows of the block table (a list of page lists) and the pool's size, in scattered order."""
    held = [_pages(t, case) for t in _lengths(case)]
    extra = 0
    if case["kind"] == "fork":
        extra = len(held) * case["samples"]
    if case["kind"] == "compact":
        extra = int(sum(held) / case["share"]) - sum(held) + 1
    total = sum(held) + extra + 3
    order = list(range(total))
    random.Random("%d %d" % (total, len(held))).shuffle(order)
    rows, at = [], 0
    for h in held:
        rows.append(order[at:at + h])
        at += h
    return rows, total


class State:
    pass


def prepare(case, seed):
    s = State()
    s.case = case
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    if case["kind"] == "prefill":
        # queries, keys and values as one projection hands them over, side by side in a row
        t, hq, hk = case["tokens"], case["heads"], case["kv_heads"]
        x = normal(t, hq + 2 * hk, D)
        x[:, :hq] *= 1.5
        x[:, hq:hq + hk] += normal(1, hk, D)  # channels of a key head have means of their own
        x = x.to(torch.bfloat16)
        s.q, s.k, s.v = x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:]
        s.offsets = _offsets(_prompt_lengths(case))
        if own:
            s.attention = _attention()
        return s

    hk, p = case["kv_heads"], case["page_tokens"]
    rows, total = _pool(case)
    layers = case.get("layers", 2)
    shape = (layers, total, 2, hk, p, D)
    values = normal(*shape) * 96.0
    values[:, :, 0] += 64.0 * normal(layers, 1, hk, 1, D)
    s.codes = values.clamp_(-CODE_MAX, CODE_MAX).to(torch.float8_e4m3fn)
    del values
    s.exponents = torch.randint(-8, -5, shape[:4], generator=g, device="cuda", dtype=torch.int8)
    sequences = len(rows) * (1 + case.get("samples", 0))
    width = max(1, max(len(r) for r in rows))
    s.table = torch.tensor([r + [0] * (width - len(r)) for r in rows]
                           + [[0] * width] * (sequences - len(rows)), dtype=torch.int32, device="cuda")
    s.lengths = torch.tensor(_lengths(case) + [0] * (sequences - len(rows)), dtype=torch.int32,
                             device="cuda")
    used = torch.zeros(total, dtype=torch.int32)
    used[[page for r in rows for page in r]] = 1
    s.references = used.cuda()
    s.width = width
    s.which = torch.arange(len(rows), dtype=torch.int32, device="cuda")
    if case["kind"] in ("attend", "append"):
        s.layer = 1
        counts = _new_rows(case)
        s.offsets, s.rows, s.most = _offsets(counts), sum(counts), max(counts)
        if case["kind"] == "attend":
            s.q = (normal(s.rows, case["heads"], D) * 0.8).to(torch.bfloat16)
        else:
            kv = (normal(s.rows, 2, hk, D) * torch.exp2(2 * normal(s.rows, 2, hk, 1))).to(torch.bfloat16)
            s.k, s.v = kv[:, 0], kv[:, 1]
    if case["kind"] == "fork":
        n, each = case["sequences"], case["samples"]
        s.parents = torch.arange(n, dtype=torch.int32, device="cuda").repeat_interleave(each)
        s.children = torch.arange(n, n * (1 + each), dtype=torch.int32, device="cuda")
    if case["kind"] == "compact":
        s.table_before, s.references_before = s.table.clone(), s.references.clone()
    if own:
        s.cache = _attention().KvCache(s.codes, s.exponents, s.table, s.lengths, s.references)
    return s


def _attention():
    return importlib.import_module("nemotron-inference_b200.attention")


def _offsets(counts):
    at = [0]
    for c in counts:
        at.append(at[-1] + c)
    return torch.tensor(at, dtype=torch.int32, device="cuda")


def run(s):
    kind = s.case["kind"]
    if kind == "prefill":
        if own:
            return s.attention.attention_prefill(s.q, s.k, s.v, s.offsets, return_lse=s.case["lse"])
        return _plain_prefill(s)
    if kind == "attend":
        return s.cache.attend(s.layer, s.q, s.which, s.offsets) if own else _plain_attend(s)
    if kind == "append":
        s.cache.append(s.layer, s.k, s.v, s.which, s.offsets) if own else _plain_append(s)
        return {"codes": s.codes, "exponents": s.exponents}
    if kind == "fork":
        s.cache.fork(s.parents, s.children) if own else _plain_fork(s)
    else:
        # the scheduler's books as they were; the pages above the dense part still hold their rows
        s.table.copy_(s.table_before)
        s.references.copy_(s.references_before)
        s.cache.compact() if own else _plain_compact(s)
    return {"codes": s.codes, "exponents": s.exponents, "table": s.table, "lengths": s.lengths,
            "references": s.references}


def _plain_prefill(s):
    """Row t sees the rows of its own sequence up to itself."""
    t, hk = s.q.shape[0], s.case["kv_heads"]
    at = torch.arange(t, device="cuda")
    sequence = torch.searchsorted(s.offsets, at.int(), right=True)
    seen = (sequence[:, None] == sequence[None, :]) & (at[None, :] <= at[:, None])
    q = s.q.float().unflatten(1, (hk, -1)).permute(1, 2, 0, 3)  # [hk, group, t, D]
    k = s.k.float().transpose(0, 1)[:, None]
    v = s.v.float().transpose(0, 1)[:, None]
    scores = (q @ k.transpose(2, 3)) * D ** -0.5
    scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(dim=3, keepdim=True)
    scores = scores.sub_(top).exp_()
    total = scores.sum(dim=3, keepdim=True)
    out = ((scores @ v) / total).permute(2, 0, 1, 3).flatten(1, 2).to(torch.bfloat16)
    if not s.case["lse"]:
        return out
    return out, (top + total.log())[..., 0].permute(2, 0, 1).flatten(1, 2).contiguous()


def _plain_attend(s):
    """New row j of a sequence stands at position length - rows + j and sees every token up to it."""
    n, hk, p = s.which.numel(), s.case["kv_heads"], s.case["page_tokens"]
    which = s.which.long()
    pages = s.table[which].long()
    values = s.codes[s.layer][pages].float()  # [n, width, 2, hk, p, D]
    values *= torch.exp2(s.exponents[s.layer][pages].float())[..., None, None]
    kv = values.permute(2, 0, 3, 1, 4, 5).flatten(3, 4)  # [2, n, hk, tokens, D]
    counts = (s.offsets[1:] - s.offsets[:-1]).long()
    held = s.lengths[which].long()
    j = torch.arange(s.most, device="cuda")
    row = (s.offsets[:-1, None].long() + j).clamp(max=s.rows - 1)
    q = s.q.float()[row].unflatten(2, (hk, -1)).transpose(1, 2)  # [n, hk, most, group, D]
    scores = (q.flatten(2, 3) @ kv[0].transpose(2, 3)) * D ** -0.5
    position = held[:, None] - counts[:, None] + j
    seen = torch.arange(s.width * p, device="cuda") <= position[..., None]  # [n, most, tokens]
    scores = scores.unflatten(2, (s.most, -1)).masked_fill(~seen[:, None, :, None], -math.inf)
    weights = (scores - scores.amax(dim=4, keepdim=True)).exp()
    out = (weights.flatten(2, 3) @ kv[1]) / weights.sum(dim=4).flatten(2, 3)[..., None]
    out = out.unflatten(2, (s.most, -1)).transpose(1, 2).flatten(2, 3)  # [n, most, heads, D]
    return out[j[None, :] < counts[:, None]].to(torch.bfloat16)


def _places(s):
    """Sequence, position, page and place in the page of every new row."""
    row = torch.arange(s.rows, device="cuda")
    i = torch.searchsorted(s.offsets, row.int(), right=True) - 1
    sequence = s.which.long()[i]
    position = s.lengths.long()[sequence] - s.offsets.long()[i + 1] + row
    p = s.case["page_tokens"]
    return sequence, position, s.table[sequence, position // p].long(), position % p


def _plain_append(s):
    """A page and head's exponent is the least that keeps its values within the codes' range."""
    _, _, page, place = _places(s)
    codes, exponents = s.codes[s.layer], s.exponents[s.layer]  # [pages, 2, hk, p, D], [pages, 2, hk]
    total, p = codes.shape[0], codes.shape[3]
    new = torch.stack([s.k, s.v], dim=1).float()  # [rows, 2, hk, D]
    top = torch.zeros_like(exponents, dtype=torch.float32)
    top.index_reduce_(0, page, new.abs().amax(dim=3), "amax")
    part, power = torch.frexp(top)
    needed = torch.where(part <= CODE_MAX / 512, power - 9, power - 8)
    needed = torch.where(top > 0, needed, EXPONENT_MIN).clamp(EXPONENT_MIN, EXPONENT_MAX)
    first = torch.full((total,), p, device="cuda").index_reduce_(0, page, place, "amin")
    before = exponents.int()
    kept = torch.maximum(before, needed)  # of a page that held tokens already
    after = torch.where((first == 0)[:, None, None], needed, kept)
    after = torch.where((first < p)[:, None, None], after, before)
    older = torch.arange(p, device="cuda") < torch.where(first < p, first, 0)[:, None]
    values = codes.float()
    lowered = values * torch.exp2((before - after).float())[..., None, None]
    values = torch.where(older[:, None, None, :, None], lowered, values)
    fit = new * torch.exp2(-after[page].float())[..., None]
    values[page, :, :, place] = fit.clamp(-CODE_MAX, CODE_MAX)
    codes.copy_(values.to(torch.float8_e4m3fn))
    exponents.copy_(after.to(torch.int8))


def _use(s, sequences):
    """Which places of these sequences' rows of the table hold pages."""
    p = s.case["page_tokens"]
    return torch.arange(s.width, device="cuda") < ((s.lengths.long()[sequences] + p - 1) // p)[:, None]


def _plain_fork(s):
    """Children share their parents' full pages and get copies of the last, partly filled ones."""
    parents, children, p = s.parents.long(), s.children.long(), s.case["page_tokens"]
    given_up = s.table[children][_use(s, children)].long()
    s.references.index_add_(0, given_up, torch.full_like(given_up, -1, dtype=torch.int32))
    lengths = s.lengths[parents]
    used = _use(s, parents)
    rows = torch.where(used, s.table[parents], 0)
    last = (lengths.long() // p)[:, None]
    partial = (lengths % p != 0).nonzero()[:, 0]
    source = rows.gather(1, last.clamp(max=s.width - 1))[partial, 0].long()
    target = (s.references == 0).nonzero()[:partial.numel(), 0]
    rows[partial, last[partial, 0]] = target.int()
    pages = rows[used].long()
    s.references.index_add_(0, pages, torch.ones_like(pages, dtype=torch.int32))
    s.table[children] = rows
    s.lengths[children] = lengths
    s.codes.view(torch.uint8)[:, target] = s.codes.view(torch.uint8)[:, source]
    s.exponents[:, target] = s.exponents[:, source]


def _plain_compact(s):
    """The i-th page in use behind the dense part moves to the i-th free one in it."""
    live = s.references > 0
    count = live.sum()
    at = torch.arange(live.numel(), device="cuda")
    source = (live & (at >= count)).nonzero()[:, 0]
    target = (~live & (at < count)).nonzero()[:, 0]
    moved = at.clone()
    moved[source] = target
    every = torch.arange(s.lengths.numel(), device="cuda")
    s.table.copy_(torch.where(_use(s, every), moved[s.table.long()].int(), s.table))
    s.references[target] = s.references[source]
    s.references[source] = 0
    s.codes.view(torch.uint8)[:, target] = s.codes.view(torch.uint8)[:, source]
    s.exponents[:, target] = s.exponents[:, source]


def work(case):
    kind = case["kind"]
    if kind == "prefill":
        t, hq, hk = case["tokens"], case["heads"], case["kv_heads"]
        pairs = sum(n * (n + 1) // 2 for n in _prompt_lengths(case))
        return {"bytes": 2 * t * D * (2 * hq + 2 * hk) + (4 * t * hq if case["lse"] else 0),
                "flops": 4 * D * hq * pairs}
    lengths, hk = _lengths(case), case["kv_heads"]
    if kind == "attend":
        counts, hq = _new_rows(case), case["heads"]
        pairs = sum(c * n - c * (c - 1) // 2 for n, c in zip(lengths, counts))
        pages = sum(_pages(n, case) for n in lengths)
        return {"bytes": 2 * hk * (D * sum(lengths) + pages) + 4 * D * hq * sum(counts),
                "flops": 4 * D * hq * pairs}
    if kind == "append":
        rows = _new_rows(case)
        pages = sum(_pages(n, case) - (n - r) // case["page_tokens"] for n, r in zip(lengths, rows))
        return {"bytes": 2 * hk * (3 * D * sum(rows) + pages), "flops": 0}
    held = [_pages(n, case) for n in lengths]
    if kind == "fork":
        copied = case["samples"] * sum(_last_is_partial(n, case) for n in lengths)
        return {"bytes": 2 * copied * _page_bytes(case) + 4 * (1 + case["samples"]) * sum(held),
                "flops": 0}
    rows, total = _pool(case)
    live = sum(held)
    moved = sum(page >= live for r in rows for page in r)
    return {"bytes": 2 * moved * _page_bytes(case) + 8 * live + 8 * total, "flops": 0}


def exact(case, seed):
    """The operators from their definitions, in 64 bits."""
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "prefill":
        return _exact_prefill(s)
    if kind == "attend":
        return _exact_attend(s)
    if kind == "append":
        return _exact_append(s)
    return None  # moves whole pages: nothing is computed


def _softmax_rows(q, k, v, seen):
    """q [rows, D], k and v [tokens, D], seen [rows, tokens] -> values [rows, D], log of the sums."""
    scores = torch.where(seen, q @ k.T / math.sqrt(D), -math.inf)
    lse = torch.logsumexp(scores, dim=1)
    return torch.exp(scores - lse[:, None]) @ v, lse


def _exact_prefill(s):
    t, hq, hk = s.case["tokens"], s.case["heads"], s.case["kv_heads"]
    out = torch.zeros((t, hq, D), dtype=torch.float64, device="cuda")
    lse = torch.zeros((t, hq), dtype=torch.float64, device="cuda")
    start = 0
    for n in _prompt_lengths(s.case):
        rows = slice(start, start + n)
        seen = torch.ones((n, n), dtype=torch.bool, device="cuda").tril()
        for h in range(hq if n else 0):
            kv = h // (hq // hk)
            out[rows, h], lse[rows, h] = _softmax_rows(
                s.q[rows, h].double(), s.k[rows, kv].double(), s.v[rows, kv].double(), seen)
        start += n
    return (out, lse) if s.case["lse"] else out


def _exact_attend(s):
    hq, hk, p = s.case["heads"], s.case["kv_heads"], s.case["page_tokens"]
    out = torch.zeros((s.rows, hq, D), dtype=torch.float64, device="cuda")
    start = 0
    for i, (n, c) in enumerate(zip(_lengths(s.case), _new_rows(s.case))):
        pages = s.table[i, :_pages(n, s.case)].long()
        scale = torch.pow(2.0, s.exponents[s.layer, pages].double())[..., None, None]
        values = s.codes[s.layer, pages].double() * scale  # [pages, 2, hk, p, D]
        at = torch.arange(n, device="cuda")
        seen = at[None, :] <= (n - c + torch.arange(c, device="cuda"))[:, None]
        for h in range(hk):
            k, v = (values[:, b, h].reshape(-1, D)[:n] for b in (0, 1))
            for x in range(h * (hq // hk), (h + 1) * (hq // hk)):
                out[start:start + c, x], _ = _softmax_rows(s.q[start:start + c, x].double(), k, v, seen)
        start += c
    return out


def _exact_append(s):
    codes, exponents = s.codes.double(), s.exponents.clone()
    hk, p = s.case["kv_heads"], s.case["page_tokens"]
    if s.rows * hk > 70000:
        return None
    start = 0
    for i, (n, c) in enumerate(zip(_lengths(s.case), _new_rows(s.case))):
        for b in range((n - c) // p, _pages(n, s.case)):
            page = int(s.table[i, b])
            first, last = max(n - c, b * p), min(n, b * p + p)  # its new tokens
            rows = slice(start + first - (n - c), start + last - (n - c))
            for half, new in ((0, s.k), (1, s.v)):
                x = new[rows].double()
                top = x.abs().amax(dim=(0, 2))
                e = torch.ceil(torch.log2(top / CODE_MAX)).clamp(EXPONENT_MIN, EXPONENT_MAX)
                less = top <= CODE_MAX * torch.exp2(e - 1)  # (a logarithm that came out too large)
                e = torch.where(less, e - 1, e).clamp(min=EXPONENT_MIN)
                held = first - b * p
                if held:
                    old = exponents[s.layer, page, half].double()
                    e = torch.maximum(e, old)
                    codes[s.layer, page, half, :, :held] = _round_code(
                        codes[s.layer, page, half, :, :held] * torch.exp2(old - e)[:, None, None])
                codes[s.layer, page, half, :, held:last - b * p] = _round_code(
                    x.transpose(0, 1) * torch.exp2(-e)[:, None, None])
                exponents[s.layer, page, half] = e.to(torch.int8)
        start += c
    return {"codes": codes, "exponents": exponents}


def _round_code(x):
    """The nearest E4M3 value, ties to the even one: steps of 1/8 of the power of two below, 2^-9 at least."""
    _, power = torch.frexp(x)
    step = torch.exp2((power - 4).clamp(min=-9).double())
    return (torch.round(x / step) * step).clamp(-CODE_MAX, CODE_MAX)
