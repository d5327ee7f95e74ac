"""Operators of long and branching streams, as cases whose time is measured.

A server that keeps many endless conversations, and answers each question several times to choose the likeliest answer,
does three things beside the model's own products:

* ``attention``: the queries of a step over a paged cache of which every query sees the last ``window`` positions and the
  sequence's first ``kept`` ones.  With s_j = scale q . k_j for the keys j of the query's own sequence that it sees
  (j <= p, and j > p - window or j < kept, p the query's position), o = sum_j exp(s_j) v_j / sum_j exp(s_j).  Pages that no
  query can see any more have been given back; the page table names the spare page in their place.
* ``logprobs``: of rows of logits x, log p_t = x_t - log sum_i exp(x_i) for a given token of each row, the entropy
  -sum_i p_i log p_i, and the ``top`` likeliest tokens with their log probabilities, equal ones by their number.
* ``copies``: a branch of a sequence shares its full pages and gets a copy of what its last page holds, in every layer;
  pages that are to be held elsewhere are moved.  ``src[i]`` goes to ``dst[i]``, its first ``tokens[i]`` positions.

Layouts are the cache's: keys [pages, kv heads, 64, head size], values transposed, [pages, kv heads, head size, 64], and
for copies a leading axis of layers.
"""
from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}
PAGE = 64
MOST_FLOPS = 2.5e11          # what a drawn step of attention may take at most
MOST_BYTES = 2.5e9           # and drawn logits and copies


def _attention(name, sequences, shortest, longest, new, heads, kv_heads, head_dim, window, kept, dtype="bfloat16"):
    """``sequences`` that hold ``shortest`` to ``longest`` tokens before the step; each brings ``new`` tokens (0: a whole
    prompt, of ``shortest`` to ``longest`` tokens, from an empty slot)."""
    return {"name": name, "op": "attention", "sequences": sequences, "shortest": shortest, "longest": longest, "new": new, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "window": window, "kept": kept, "dtype": dtype}


def _logprobs(name, rows, vocab, top, rounded=False):
    """``rounded``: the logits have passed through bfloat16, so that many are equal."""
    return {"name": name, "op": "logprobs", "rows": rows, "vocab": vocab, "top": top, "rounded": rounded}


def _copies(name, layers, sources, branches, tokens, kv_heads, head_dim, dtype="bfloat16"):
    """``sources`` pages, each copied to ``branches`` others; ``tokens`` of their positions, 0: as many as it happens."""
    return {"name": name, "op": "copies", "layers": layers, "sources": sources, "branches": branches, "tokens": tokens, "kv_heads": kv_heads,
            "head_dim": head_dim, "dtype": dtype}


def listed():
    return [
        # a single long chat's next token: latency
        _attention("decode_1", 1, 5000, 5000, 1, 32, 8, 128, 2048, 4),
        # a server's batch of chats of all lengths, most of them longer than the window
        _attention("decode_48_ragged", 48, 300, 9000, 1, 32, 8, 128, 4096, 4),
        # a few questions of unequal lengths that arrived together
        _attention("prompts_4_ragged", 4, 50, 2100, 0, 40, 8, 128, 1024, 4),
        # a turn's new tokens behind a long history, small heads, kept positions that end inside a page
        _attention("piece_517_behind_6000", 1, 6000, 6000, 517, 16, 4, 64, 1000, 100),
        # a long document from its first token on
        _attention("prompt_8192", 1, 8192, 8192, 0, 32, 8, 128, 2048, 64),
        # the 32-bit mode, in which results are checked
        _attention("prompt_157_float32", 1, 157, 157, 0, 32, 8, 128, 64, 4, "float32"),
        # one user's chat that shows each token's alternatives
        _logprobs("logprobs_1", 1, 151936, 20),
        # a batch's drawn tokens, with a few alternatives each; logits that have passed through bfloat16
        _logprobs("logprobs_48", 48, 151936, 5, True),
        # a document is scored: every position's token and the entropy, no alternatives
        _logprobs("logprobs_2047", 2047, 151936, 0),
        # one more answer to a question: a copy of the last page's 37 positions in all layers
        _copies("fork_1", 36, 1, 1, 37, 8, 128),
        # eight answers to each of six questions of any length
        _copies("fork_6_by_8", 36, 6, 8, 0, 8, 128),
        # a pool's pages moved together
        _copies("move_120", 36, 120, 1, 64, 8, 128),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "logprobs", "copies"])
    if op == "logprobs":
        vocab = rng.choice([151936, 151936, _spread(rng, 1000, 260000)])
        return _unnamed(_logprobs("", _spread(rng, 1, max(1, int(MOST_BYTES / 2 / (4 * vocab)))), vocab, rng.choice([0, 0, 1, 5, 20, rng.randint(1, 64)]), rng.random() < 0.3))
    dtype = "float32" if rng.random() < 0.15 else "bfloat16"
    if op == "copies":
        layers, kv_heads, head_dim = rng.choice([1, 28, 36, 40, 64, rng.randint(1, 64)]), rng.choice([1, 2, 4, 8, 8]), rng.choice([64, 128, 128])
        page = 2 * layers * kv_heads * PAGE * head_dim * DTYPES[dtype].itemsize
        branches = _spread(rng, 1, 16)
        sources = min(_spread(rng, 1, 128), max(1, int(MOST_BYTES / page / (1 + branches))))
        return _unnamed(_copies("", layers, sources, branches, rng.choice([0, 0, 64, rng.randint(1, 64)]), kv_heads, head_dim, dtype))
    heads, kv_heads, head_dim = rng.choice([(32, 8, 128), (32, 8, 128), (40, 8, 128), (64, 8, 128), (16, 4, 64), (8, 8, 64), (16, 2, 128)])
    kind = rng.choice(["decode", "decode", "prompt", "piece"])
    sequences = _spread(rng, 1, 64) if kind == "decode" else _spread(rng, 1, 6)
    longest = _spread(rng, 64, 16000)
    shortest = longest if rng.random() < 0.3 else rng.randint(max(1, longest // 8), longest)
    new = {"decode": 1, "prompt": 0, "piece": _spread(rng, 2, 2048)}[kind]
    case = _attention("", sequences, shortest, longest, new, heads, kv_heads, head_dim, _spread(rng, 64, 8192), _spread(rng, 1, 300), dtype)
    # (the 32-bit mode is one for checks: short and few)
    few = 2e9 if dtype == "float32" and kind != "decode" else MOST_FLOPS
    while work(case)["flops"] > few or work(case)["bytes"] > MOST_BYTES or _scores(case) > 2.2e9:
        case["longest"] = max(8, case["longest"] * 3 // 4)
        case["shortest"] = min(case["shortest"], case["longest"])
        case["sequences"] = max(1, case["sequences"] * 7 // 8)
        case["new"] = case["new"] if case["new"] < 2 else max(2, case["new"] * 3 // 4)
    return _unnamed(case)


def _unnamed(case):
    del case["name"]
    return case


# ---- what a case's sequences are ----------------------------------------------------------------------------------

def _lengths(case):
    """(tokens before the step, new tokens) of each sequence, spread evenly between the shortest and the longest."""
    n, low, high = case["sequences"], case["shortest"], case["longest"]
    held = [high if n == 1 else low + round((high - low) * ((i * 0.6180339887 + 0.5) % 1.0)) for i in range(n)]
    return [(h, case["new"]) if case["new"] else (0, h) for h in held]


def _scores(case):
    """Scores that the plain form holds at once."""
    lengths = _lengths(case)
    new, total = max(n for _, n in lengths), max(s + n for s, n in lengths)
    return case["sequences"] * case["heads"] * new * min(total, case["window"] - 1 + new + case["kept"])


def _seen(p, window, kept):
    """How many keys a query at position p sees."""
    return min(p + 1, window) + min(kept, max(0, p + 1 - window))


def work(case):
    if case["op"] == "logprobs":
        n, v, top = case["rows"], case["vocab"], case["top"]
        return {"bytes": 4 * n * v + 12 * n + 8 * n * top, "flops": 5 * n * v}
    if case["op"] == "copies":
        at = case["layers"] * case["kv_heads"] * case["head_dim"] * DTYPES[case["dtype"]].itemsize * 2
        held = _held(case)
        return {"bytes": at * sum(held) * (1 + case["branches"]), "flops": 0}
    window, kept, row = case["window"], case["kept"], case["head_dim"] * DTYPES[case["dtype"]].itemsize
    keys = pairs = queries = 0
    for start, new in _lengths(case):
        first = max(0, start - window + 1)
        keys += start + new - first + min(kept, first)
        pairs += sum(_seen(p, window, kept) for p in range(start, start + new))
        queries += new
    return {"bytes": 2 * row * (case["kv_heads"] * keys + case["heads"] * queries), "flops": 4 * case["head_dim"] * case["heads"] * pairs}


def _held(case):
    """Positions that each source page holds."""
    return [case["tokens"] or 1 + (i * 37 + 20) % PAGE for i in range(case["sources"])]


# ---- inputs -------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    return {"attention": _prepare_attention, "logprobs": _prepare_logprobs, "copies": _prepare_copies}[case["op"]](case, g)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _prepare_attention(case, g):
    dtype, window, kept = DTYPES[case["dtype"]], case["window"], case["kept"]
    lengths = _lengths(case)
    kept_pages = (kept + PAGE - 1) // PAGE
    lists = []
    for start, new in lengths:
        pages, first = (start + new + PAGE - 1) // PAGE, max(0, start - window + 1) // PAGE
        lists.append([p for p in range(pages) if p < kept_pages or p >= first])
    n_pages, width = sum(len(x) for x in lists), max((s + n + PAGE - 1) // PAGE for s, n in lengths)
    order = torch.randperm(n_pages, device=DEVICE, generator=g).tolist()        # a sequence's pages lie anywhere in the pool
    slots = torch.randperm(len(lengths) + 2, device=DEVICE, generator=g).tolist()[:len(lengths)]
    table = torch.full((len(lengths) + 2, width), n_pages, dtype=torch.int32)    # the spare page behind the others
    for slot, pages in zip(slots, lists):
        table[slot, pages] = torch.tensor([order.pop() for _ in pages], dtype=torch.int32)
    cu = [0]
    for _, new in lengths:
        cu.append(cu[-1] + new)

    def normal(*shape):
        return torch.randn(shape, device=DEVICE, generator=g, dtype=torch.float32).to(dtype)
    hkv, hd = case["kv_heads"], case["head_dim"]
    return {"op": "attention", "q": normal(cu[-1], case["heads"] * hd) * 2, "k": normal(n_pages + 1, hkv, PAGE, hd), "v": normal(n_pages + 1, hkv, hd, PAGE),
            "table": table.to(DEVICE), "slot": _ints(slots), "start": _ints([s for s, _ in lengths]), "new": _ints([n for _, n in lengths]), "cu": _ints(cu),
            "max_new": max(n for _, n in lengths), "max_total": max(s + n for s, n in lengths), "heads": case["heads"], "kv_heads": hkv, "head_dim": hd,
            "scale": hd ** -0.5, "window": window, "kept": kept}


def _prepare_logprobs(case, g):
    n, v = case["rows"], case["vocab"]
    x = torch.randn((n, v), device=DEVICE, generator=g).mul_(2.5)
    # a model is often sure: some rows have a few tokens far above the others
    likely = torch.randint(0, v, (n, 8), device=DEVICE, generator=g)
    x.scatter_add_(1, likely, torch.rand((n, 8), device=DEVICE, generator=g) * torch.rand((n, 1), device=DEVICE, generator=g) * 25.0)
    if case["rounded"]:
        x = x.bfloat16().float()
    return {"op": "logprobs", "logits": x, "tokens": likely[:, 0].to(torch.int32).contiguous(), "top": case["top"]}


def _prepare_copies(case, g):
    sources, branches = case["sources"], case["branches"]
    pages = sources * (1 + branches)
    order = torch.randperm(pages, device=DEVICE, generator=g).tolist()
    src = [order[i] for i in range(sources) for _ in range(branches)]
    tokens = [n for n in _held(case) for _ in range(branches)]
    layers, hkv, hd, dtype = case["layers"], case["kv_heads"], case["head_dim"], DTYPES[case["dtype"]]
    k = torch.empty((layers, pages + 1, hkv, PAGE, hd), dtype=dtype, device=DEVICE).normal_(generator=g)
    v = torch.empty((layers, pages + 1, hkv, hd, PAGE), dtype=dtype, device=DEVICE).normal_(generator=g)
    return {"op": "copies", "k": k, "v": v, "src": src, "dst": order[sources:], "tokens": tokens}


# ---- one pass -----------------------------------------------------------------------------------------------------

def run(state):
    s = state
    if own:
        from palm_infra_amd.kernels import ops
        if s["op"] == "attention":
            return ops.attention_kept(s["q"], s["k"], s["v"], s["table"], s["slot"], s["start"], s["new"], s["cu"], s["max_new"], s["max_total"],
                                      s["heads"], s["kv_heads"], s["head_dim"], s["scale"], s["window"], s["kept"])
        if s["op"] == "logprobs":
            return ops.token_logprobs(s["logits"], s["tokens"], s["top"])
        ops.copy_pages(s["k"], s["v"], s["src"], s["dst"], s["tokens"])
        return s["k"], s["v"]
    return {"attention": _plain_attention, "logprobs": _plain_logprobs, "copies": _plain_copies}[s["op"]](s)


def _plain_attention(s):
    nh, hkv, hd, window, kept, max_new, total = (s[x] for x in ("heads", "kv_heads", "head_dim", "window", "kept", "max_new", "max_total"))
    q, start, new, cu = s["q"], s["start"].long(), s["new"].long(), s["cu"].long()
    B = start.shape[0]
    # the positions that a sequence's queries see: its first ones, then those from the first query's window on
    span = min(total, window - 1 + max_new)
    first = (start - window + 1).clamp(min=0)
    head = torch.arange(min(kept, total), device=q.device).expand(B, -1)
    rest = first[:, None] + torch.arange(span, device=q.device)
    at = torch.cat([head, rest], 1)                                             # [B, C]
    there = torch.cat([head < first[:, None], rest < (start + new)[:, None]], 1)
    at = torch.where(there, at, 0)
    pages = s["table"].long()[s["slot"].long()].gather(1, at // PAGE)
    k = s["k"][pages, :, at % PAGE].float().permute(0, 2, 1, 3).contiguous()    # [B, kv heads, C, head size]
    v = s["v"][pages, :, :, at % PAGE].float().permute(0, 2, 1, 3).contiguous()
    i = torch.arange(max_new, device=q.device)
    pos = start[:, None] + i                                                    # [B, new]
    rows = (cu[:-1, None] + torch.minimum(i, (new - 1).clamp(min=0)[:, None]))
    g = nh // hkv
    x = q[rows].float().view(B, max_new, hkv, g, hd).permute(0, 2, 3, 1, 4).reshape(B, hkv, g * max_new, hd)
    scores = torch.matmul(x, k.transpose(2, 3)).mul_(s["scale"]).view(B, hkv, g, max_new, at.shape[1])
    key, p = at[:, None, :], pos[:, :, None]
    seen = there[:, None, :] & (key <= p) & ((key > p - window) | (key < kept))
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    total_weight = scores.sum(-1, keepdim=True)
    o = torch.matmul(scores.view(B, hkv, g * max_new, -1), v).view(B, hkv, g, max_new, hd) / total_weight
    o = o.permute(0, 3, 1, 2, 4).reshape(B, max_new, nh * hd)
    row = torch.arange(q.shape[0], device=q.device)
    b = torch.searchsorted(cu, row, right=True) - 1
    return o[b, row - cu[b]].to(q.dtype)


def _plain_logprobs(s):
    x, top = s["logits"], s["top"]
    n, v = x.shape
    t = x - x.amax(1, keepdim=True)
    e = t.exp()
    total = e.sum(1, dtype=torch.float64)                                       # (a long sum)
    log_total = total.log()
    entropy = log_total - torch.where(e > 0, t * e, 0).sum(1, dtype=torch.float64) / total
    tokens = s["tokens"].long()
    given = t.gather(1, tokens.clamp(0, v - 1)[:, None])[:, 0].double() - log_total
    given = torch.where((tokens >= 0) & (tokens < v), given, math.nan)
    # by value, then by number: the bits of a float are in its order where it is positive, and in the other where it is not
    bits = (x + 0.0).view(torch.int32).long()
    order = torch.where(bits < 0, -(bits & 0x7fffffff), bits)
    ids = ((order << 32) - torch.arange(v, device=x.device)).topk(top, dim=1).indices
    return given.float(), entropy.float(), ids.to(torch.int32), (t.gather(1, ids).double() - log_total[:, None]).float()


def _plain_copies(s):
    k, v = s["k"], s["v"]
    src, dst = (torch.tensor(s[x], device=k.device) for x in ("src", "dst"))
    filled = torch.arange(PAGE, device=k.device) < torch.tensor(s["tokens"], device=k.device)[:, None]
    k[:, dst] = torch.where(filled[:, None, :, None], k[:, src], k[:, dst])
    v[:, dst] = torch.where(filled[:, None, None, :], v[:, src], v[:, dst])
    return k, v


# ---- the same in 64 bits ------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "logprobs":
        return _exact_logprobs(s)
    if case["op"] == "attention":
        return _exact_attention(s)
    k, v = s["k"].double(), s["v"].double()
    for src, dst, n in zip(s["src"], s["dst"], s["tokens"]):
        k[:, dst, :, :n] = s["k"][:, src, :, :n].double()
        v[:, dst, :, :, :n] = s["v"][:, src, :, :, :n].double()
    return k, v


def _exact_logprobs(s):
    given, entropy, ids, best = [], [], [], []
    for row, token in zip(s["logits"], s["tokens"].tolist()):
        x = row.double()
        logp = x - torch.logsumexp(x, 0)
        given.append(logp[token])
        entropy.append(-(logp.exp() * logp).sum())
        likeliest = torch.sort(x, descending=True, stable=True).indices[:s["top"]] if s["top"] else torch.zeros((0,), dtype=torch.long, device=x.device)
        ids.append(likeliest)
        best.append(logp[likeliest])
    return torch.stack(given), torch.stack(entropy), torch.stack(ids).to(torch.int32), torch.stack(best)


def _exact_attention(s):
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEVICE)
    nh, hd, group = s["heads"], s["head_dim"], s["heads"] // s["kv_heads"]
    for slot, start, new, row in zip(s["slot"].tolist(), s["start"].tolist(), s["new"].tolist(), s["cu"].tolist()):
        for lo in range(0, new, 2048):                                          # queries at a time
            n = min(2048, new - lo)
            p = torch.arange(start + lo, start + lo + n, device=DEVICE)[:, None]
            begin = max(0, start + lo - s["window"] + 1)
            j = torch.tensor(list(range(min(s["kept"], begin))) + list(range(begin, start + lo + n)), device=DEVICE)
            hidden = (j > p) | ((j <= p - s["window"]) & (j >= s["kept"]))
            page = s["table"][slot].long()[j // PAGE]
            for h in range(nh):
                q = s["q"][row + lo:row + lo + n, h * hd:(h + 1) * hd].double()
                k, v = s["k"][page, h // group, j % PAGE].double(), s["v"][page, h // group, :, j % PAGE].double()
                weights = torch.softmax((q @ k.T * s["scale"]).masked_fill(hidden, -math.inf), 1)
                out[row + lo:row + lo + n, h * hd:(h + 1) * hd] = weights @ v
    return out
