"""Several answers to one prompt: log probabilities of tokens, and the pages of a cache that the answers share.

Five operators, each as a plain form (elementary torch operations) and as the framework's own call:

  token_logprobs   logits -> log p of given tokens, entropy of the row, its k most probable tokens
  linear_logprobs  hidden states and LM-head weight -> log p of given tokens and entropy, no logits kept
  copy_pages       pages of a paged KV cache onto other pages, in every layer
  fork             rows of a block table continue others (beams, parallel answers): the pages are shared and
                   counted, and the last page, where rows would write into one another, becomes private
  compact          some rows give their pages back, the others' pages move to the front of the cache

A row of logits x has p_i = exp(x_i - m) / S, m = max x, S = sum exp(x_i - m); entropy = ln S - sum p_i (x_i - m).
A row that its mask leaves empty (all -inf) has log p = -inf and entropy 0; tokens of probability 0 are no
alternatives (id -1, log p -inf); a token id of -1 asks for nothing and gets 0.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
ROW = 576    # latent KV row: 512 latent + 64 rope dims
BLOCK = 64   # tokens of a page


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one user's decode step that asks for its token and five alternatives: latency
        dict(name="logprobs 1 row", op="token_logprobs", rows=1, vocab=102400, dtype="bf16", given=1, top_k=5, pad=0, mask=""),
        # a decode step of 64 requests with the most alternatives that the chat API allows
        dict(name="logprobs 64 rows", op="token_logprobs", rows=64, vocab=102400, dtype="bf16", given=1, top_k=20, pad=0, mask=""),
        # constrained decoding of a verify round, fp32 logits: a grammar's mask leaves few tokens, or none; four
        # choices are scored; odd sizes and strides
        dict(name="logprobs masked fp32", op="token_logprobs", rows=515, vocab=129281, dtype="fp32", given=4, top_k=8, pad=7, mask="grammar"),
        # a whole prefill chunk: every prompt token's log probability and alternatives
        dict(name="logprobs 8192 rows", op="token_logprobs", rows=8192, vocab=102400, dtype="bf16", given=1, top_k=20, pad=0, mask=""),
        # a small batch scored straight from its hidden states, ragged: the LM head's weight is read once
        dict(name="linear 61 rows ragged", op="linear_logprobs", rows=61, vocab=102397, hidden=2048),
        # a whole prefill chunk of a prompt that is scored
        dict(name="linear 8192 rows", op="linear_logprobs", rows=8192, vocab=102400, hidden=2048),
        # pages handed from one sequence to another, bf16 and fp8 caches
        dict(name="copy 3 pages fp8", op="copy_pages", layers=27, pages=64, copies=3, cache="fp8"),
        dict(name="copy 400 pages", op="copy_pages", layers=27, pages=1024, copies=400, cache="bf16"),
        # a beam step of one request
        dict(name="fork 4 beams", op="fork", layers=27, pages=256, groups=1, width=4, children=4, context=1000, cache="bf16"),
        # 64 prompts that get four answers each
        dict(name="fork 64 to 256 rows", op="fork", layers=27, pages=2048, groups=64, width=1, children=4, context=1310, cache="fp8"),
        # the answers that lost give their pages back, the rest moves together: one request's, and a whole batch's
        dict(name="compact 64 pages fp8", op="compact", layers=27, pages=64, rows=4, kept=2, row_pages=12, moved=9, cache="fp8"),
        dict(name="compact 1024 pages", op="compact", layers=27, pages=1024, rows=48, kept=30, row_pages=20, moved=250, cache="bf16"),
    ]


def draw(rng):
    def log(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    op = rng.choice(["token_logprobs", "linear_logprobs", "copy_pages", "fork", "compact"])
    if op == "token_logprobs":
        vocab = log(300, 163840)
        return dict(op=op, rows=log(1, min(8192, 400_000_000 // vocab)), vocab=vocab, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                    given=rng.choice([1, 1, 4, 9]), top_k=rng.choice([0, 1, 5, 20, 32]), pad=rng.choice([0, 0, 8, 13]),
                    mask=rng.choice(["", "", "grammar", "lowest"]))
    if op == "linear_logprobs":
        vocab, hidden = log(300, 163840), 8 * log(8, 896)
        return dict(op=op, rows=log(1, max(1, min(8192, 1_500_000_000_000 // (2 * vocab * hidden)))), vocab=vocab, hidden=hidden)
    cache, layers = rng.choice(["bf16", "fp8"]), log(1, 61)
    if op == "copy_pages":
        copies = log(1, max(1, 12000 // layers))
        return dict(op=op, layers=layers, pages=2 * copies + rng.randrange(1, 40), copies=copies, cache=cache)
    if op == "fork":
        groups, width, children, context = log(1, 64), rng.choice([1, 1, 2, 4, 8]), rng.choice([1, 2, 4, 8]), log(1, 1500)
        need = groups * (width * -(-context // BLOCK) + children * 2) + rng.randrange(1, 30)
        layers = max(1, min(layers, 50000 // need))
        return dict(op=op, layers=layers, pages=need, groups=groups, width=width, children=children, context=context, cache=cache)
    rows, row_pages = log(2, 128), log(1, 40)
    kept = rng.randrange(1, rows)
    pages = rows * row_pages + rng.randrange(0, 100)
    live = kept * row_pages
    layers = max(1, min(layers, 30000 // pages))
    return dict(op=op, layers=layers, pages=pages, rows=rows, kept=kept, row_pages=row_pages,
                moved=rng.randrange(0, min(live, pages - live) + 1), cache=cache)


def _page_bytes(case):
    return case["layers"] * BLOCK * (ROW * 2 if case["cache"] == "bf16" else ROW + 5 * 4)


def _beams(case):
    """Lengths of the rows that are there and the row that each new row continues, from the case alone: some rows
    have several successors, some none."""
    groups, width, children, context = case["groups"], case["width"], case["children"], case["context"]
    lens = [max(1, context - 37 * b % (context // 8 + 1)) for b in range(groups * width)]
    parents = [g * width + i * i % width for g in range(groups) for i in range(children)]
    return lens, parents


def work(case):
    if case["op"] == "token_logprobs":
        size = 4 if case["dtype"] == "fp32" else 2
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size + case["rows"] * (8 * case["given"] + 4 + 8 * case["top_k"]), "flops": 4 * n}
    if case["op"] == "linear_logprobs":
        t, v, h = case["rows"], case["vocab"], case["hidden"]
        return {"bytes": 2 * (t * h + v * h) + 12 * t, "flops": 2 * t * v * h}
    if case["op"] == "copy_pages":
        return {"bytes": 2 * case["copies"] * _page_bytes(case), "flops": 0}
    if case["op"] == "fork":
        lens, parents = _beams(case)
        copied = sum(lens[p] % BLOCK for i, p in enumerate(parents) if p in parents[i + 1:])
        entries = (len(lens) + 2 * len(parents)) * (case["context"] // BLOCK + 2) + 2 * case["pages"]
        return {"bytes": 2 * copied * _page_bytes(case) // BLOCK + 4 * entries, "flops": 0}
    return {"bytes": 2 * case["moved"] * _page_bytes(case) + 8 * (case["rows"] * case["row_pages"] + 2 * case["pages"]), "flops": 0}


# ------------------------------------------------------------------ inputs
def _cache(case, g):
    """Latent rows of every layer; the fp8 cache holds e4m3 rows and a scale for each 128 elements."""
    slots = case["pages"] * BLOCK
    data = torch.randn(case["layers"], slots, ROW, device="cuda", dtype=torch.bfloat16, generator=g)
    if case["cache"] == "bf16":
        return data, None
    scales = torch.rand(case["layers"], slots, 5, device="cuda", generator=g) * 0.01 + 1e-4
    return data.to(torch.float8_e4m3fn).view(torch.uint8), scales


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    if case["op"] == "token_logprobs":
        rows, vocab, dtype = case["rows"], case["vocab"], DTYPES[case["dtype"]]
        x = torch.randn(rows, vocab + case["pad"], device="cuda", generator=g) * 2.5
        # what a model is sure of: a few tokens of each row stand out
        named = vocab - vocab // 50 if case["mask"] == "lowest" else vocab
        sure = torch.randint(0, named, (rows, 6), device="cuda", generator=g)
        x.scatter_add_(1, sure, torch.rand(rows, 6, device="cuda", generator=g) * 9.0)
        ids = torch.randint(0, named, (rows, case["given"]), device="cuda", generator=g)
        ids[:, 0] = torch.where(torch.rand(rows, device="cuda", generator=g) < 0.8, sure[:, 0], ids[:, 0])
        x = x.to(dtype)
        row = torch.arange(rows, device="cuda")
        if case["mask"] == "grammar":
            left = torch.rand(rows, 1, device="cuda", generator=g) ** 4   # the share of tokens that a row's grammar allows
            x[torch.rand(x.shape, device="cuda", generator=g) > left] = float("-inf")
            x[row % 11 == 5] = float("-inf")
            ids[row % 7 == 3] = -1
        if case["mask"] == "lowest":
            x[:, vocab - vocab // 50:] = torch.finfo(dtype).min
            x[row % 101 == 50] = torch.finfo(dtype).min
        s["logits"] = x[:, :vocab]
        s["ids"] = ids.int() if case["given"] > 1 else ids[:, 0].int()
    elif case["op"] == "linear_logprobs":
        rows, vocab, hidden = case["rows"], case["vocab"], case["hidden"]
        s["x"] = torch.randn(rows, hidden, device="cuda", generator=g).bfloat16()
        s["w"] = (torch.randn(vocab, hidden, device="cuda", generator=g) * (2.5 / math.sqrt(hidden))).bfloat16()
        s["ids"] = torch.randint(0, vocab, (rows,), device="cuda", generator=g).int()
    else:
        s["data"], s["scales"] = _cache(case, g)
        order = torch.randperm(case["pages"], device="cuda", generator=g).int()
        if case["op"] == "copy_pages":
            n = case["copies"]
            s["src"], s["dst"] = order[:n].clone(), order[n:2 * n].clone()
        elif case["op"] == "fork":
            lens, parents = _beams(case)
            cols = case["context"] // BLOCK + 2
            s["lens"], s["parents"] = _ints(lens), _ints(parents)
            used = (s["lens"] + BLOCK - 1) // BLOCK
            col = torch.arange(cols, device="cuda")
            held = col < used[:, None]
            at = (torch.cumsum(used, 0) - used)[:, None] + col
            s["table"] = torch.where(held, order[at.clamp(max=case["pages"] - 1)], -1).int()
            s["refs"] = torch.zeros(case["pages"], dtype=torch.int32, device="cuda")
            s["refs"][s["table"][held].long()] = 1
        else:
            # the kept rows' pages: all but `moved` of them are in the part of the cache where they end up
            live, moved = case["kept"] * case["row_pages"], case["moved"]
            low = torch.randperm(live, device="cuda", generator=g)[:live - moved]
            high = live + torch.randperm(case["pages"] - live, device="cuda", generator=g)[:moved]
            mine = torch.cat([low, high])[torch.randperm(live, device="cuda", generator=g)]
            rest = torch.ones(case["pages"], dtype=torch.bool, device="cuda")
            rest[mine] = False
            rest = rest.nonzero()[:, 0]
            lost = (case["rows"] - case["kept"]) * case["row_pages"]
            table = torch.cat([mine, rest[torch.randperm(rest.numel(), device="cuda", generator=g)][:lost]])
            table = table.view(case["rows"], case["row_pages"])
            where = torch.randperm(case["rows"], device="cuda", generator=g)
            s["table"] = torch.full((case["rows"], case["row_pages"] + 1), -1, dtype=torch.int32, device="cuda")
            s["table"][where, :case["row_pages"]] = table.int()
            s["lost"] = where[case["kept"]:].int()
            s["refs"] = torch.zeros(case["pages"], dtype=torch.int32, device="cuda")
            s["refs"][table.reshape(-1)] = 1
    return s


# ------------------------------------------------------------------ plain forms
def plain_token_logprobs(logits, ids, top_k):
    x = logits.float() + 0.0
    vocab = x.shape[1]
    top = x.amax(1, keepdim=True)
    m = torch.where(top == float("-inf"), 0.0, top)
    t = x - m
    p = torch.exp(t)
    total = p.sum(1, dtype=torch.float64)
    mean = torch.where(p > 0, p * t, 0.0).sum(1, dtype=torch.float64)
    log_total = torch.log(total)
    bad = torch.isnan(total)
    empty = total == 0
    entropy = torch.where(empty, 0.0, log_total - mean / total)
    shift = torch.where(empty, 0.0, log_total)
    at = ids.view(ids.shape[0], -1).long()
    given = torch.gather(t, 1, at.clamp(0, vocab - 1)).double() - shift[:, None]
    given = torch.where(at == -1, 0.0, torch.where((at < 0) | (at >= vocab), float("nan"), given))
    # larger logit first, then lower id: both in one whole number
    bits = x.view(torch.int32).long()
    order = torch.where(bits < 0, -2147483648 - bits, bits)
    key = torch.topk((order << 32) + (vocab - 1 - torch.arange(vocab, device=x.device)), top_k, dim=1).values
    best = vocab - 1 - (key & 0xFFFFFFFF)
    value = torch.gather(t, 1, best).double() - shift[:, None]
    none = (value == float("-inf")) | bad[:, None]
    value = torch.where(bad[:, None], float("nan"), value)
    return given.float().view(ids.shape), entropy.float(), value.float(), torch.where(none, -1, best).int()


def plain_linear_logprobs(x, w, ids):
    logits = x.float() @ w.float().t()
    m = logits.amax(1, keepdim=True)
    t = logits - m
    p = torch.exp(t)
    total = p.sum(1, dtype=torch.float64)
    entropy = torch.log(total) - (p * t).sum(1, dtype=torch.float64) / total
    given = torch.gather(t, 1, ids.long().clamp(min=0)[:, None])[:, 0].double() - torch.log(total)
    return torch.where(ids < 0, 0.0, given).float(), entropy.float()


def plain_copy_rows(plane, src, dst):
    if plane is not None:
        plane[:, dst] = plane[:, src]


def plain_pages(plane, pages):
    return None if plane is None else plane.view(plane.shape[0], pages, -1)


def plain_copy_pages(data, scales, pages, src, dst):
    ok = (src >= 0) & (src < pages) & (dst >= 0) & (dst < pages)
    src, dst = src[ok].long(), dst[ok].long()
    plain_copy_rows(plain_pages(data, pages), src, dst)
    plain_copy_rows(plain_pages(scales, pages), src, dst)


def plain_count(refs, table, by):
    """refs[p] += by for every entry p of the table; entries that are no page count nowhere."""
    held = (table >= 0) & (table < refs.numel())
    counts = torch.zeros(refs.numel() + 1, dtype=torch.int32, device=refs.device)
    counts.index_add_(0, torch.where(held, table, refs.numel()).reshape(-1), torch.full((table.numel(),), by, dtype=torch.int32, device=refs.device))
    refs += counts[:-1]


def plain_fork(table, lens, parents, refs):
    rows, cols = table.shape
    there = (parents >= 0) & (parents < rows)
    of = parents.clamp(0, rows - 1).long()
    new_lens = torch.where(there, lens[of], 0)
    held = torch.arange(cols, device=table.device) < ((new_lens + BLOCK - 1) // BLOCK)[:, None]
    new_table = torch.where(held, table[of], -1)
    plain_count(refs, table, -1)
    plain_count(refs, new_table, 1)
    return new_table, new_lens


def plain_reserve(table, lens, refs, data, scales, tokens):
    """Room for `tokens` more tokens in every row that has any, from the lowest free pages, row by row."""
    rows, cols = table.shape
    pages = refs.numel()
    want = torch.where(lens > 0, tokens, 0)
    col = torch.arange(cols, device=table.device)
    fresh = (col >= ((lens + BLOCK - 1) // BLOCK)[:, None]) & (col < ((lens + want + BLOCK - 1) // BLOCK)[:, None]) & (table < 0)
    tail_col = (lens // BLOCK).clamp(max=cols - 1).long()[:, None]
    tail = torch.gather(table, 1, tail_col)[:, 0]
    partial = (want > 0) & (lens % BLOCK != 0) & (lens // BLOCK < cols) & (tail >= 0) & (tail < pages)
    same = (tail[:, None] == tail[None, :]) & partial[:, None] & partial[None, :]
    before = torch.tril(same, -1).sum(1)
    own_page = tail.clamp(0, pages - 1).long()
    private = partial & (refs[own_page] - before > 1)
    need = private.int() + fresh.sum(1, dtype=torch.int32)
    start = torch.cumsum(need, 0) - need
    free = refs <= 0
    served = (start + need <= free.sum()) & (need > 0)
    short = torch.where(served, 0, need).int()
    order = torch.argsort(torch.where(free, 0, 1), stable=True)
    grant = order[(start[:, None] + private[:, None] + torch.cumsum(fresh, 1) - 1).clamp(0, pages - 1)]
    fresh &= served[:, None]
    private &= served
    copy = order[start.clamp(max=pages - 1)]
    # private copies: the tokens that the row has in its last page
    row = torch.arange(BLOCK, device=table.device)
    moved = (private[:, None] & (row < (lens % BLOCK)[:, None]))
    src, dst = (own_page[:, None] * BLOCK + row)[moved], (copy[:, None] * BLOCK + row)[moved]
    plain_copy_rows(data, src, dst)
    plain_copy_rows(scales, src, dst)
    table.copy_(torch.where(fresh, grant, table))
    table.scatter_(1, tail_col, torch.where(private, copy, torch.gather(table, 1, tail_col)[:, 0]).int()[:, None])
    plain_count(refs, torch.where(private, tail, -1), -1)
    plain_count(refs, torch.where(private, copy, -1), 1)
    plain_count(refs, torch.where(fresh, grant, -1), 1)
    return short


def plain_free(table, refs, rows):
    gone = torch.zeros(table.shape[0] + 1, dtype=torch.bool, device=table.device)
    gone[torch.where((rows >= 0) & (rows < table.shape[0]), rows, table.shape[0]).long()] = True
    plain_count(refs, torch.where(gone[:-1, None], table, -1), -1)
    table.masked_fill_(gone[:-1, None], -1)


def plain_compact(table, refs, data, scales):
    pages = refs.numel()
    page = torch.arange(pages, device=refs.device)
    live = refs > 0
    count = live.sum()
    holes = torch.nonzero(~live & (page < count))[:, 0]
    moving = torch.nonzero(live & (page >= count))[:, 0]
    plain_copy_rows(plain_pages(data, pages), moving, holes)
    plain_copy_rows(plain_pages(scales, pages), moving, holes)
    page_map = torch.where(live, page, -1).int()
    page_map[moving] = holes.int()
    held = (table >= 0) & (table < pages)
    table.copy_(torch.where(held, page_map[table.clamp(0, pages - 1).long()], table))
    moved = refs[moving]
    refs[moving] = 0
    refs[holes] = moved
    return page_map, count.int().view(1)


# ------------------------------------------------------------------ one pass
def _values(data, scales):
    """The cache as the values that it holds."""
    return (data,) if scales is None else (data.view(torch.float8_e4m3fn), scales)


def run(s):
    if own:
        from sparkpipe_rs_b200 import ops
    op = s["op"]
    if op == "token_logprobs":
        if own:
            return tuple(ops.token_logprobs(s["logits"], s["ids"], top_k=s["top_k"]))
        return plain_token_logprobs(s["logits"], s["ids"], s["top_k"])
    if op == "linear_logprobs":
        if own:
            return tuple(ops.linear_logprobs(s["x"], s["w"], s["ids"]))
        return plain_linear_logprobs(s["x"], s["w"], s["ids"])
    data, scales, pages = s["data"], s["scales"], s["pages"]
    if op == "copy_pages":
        if own:
            ops.copy_pages(data, s["src"], s["dst"], cache_scales=scales)
        else:
            plain_copy_pages(data, scales, pages, s["src"], s["dst"])
        return _values(data, scales)
    refs = s["refs"].clone()
    if op == "fork":
        if own:
            table, lens = ops.fork_pages(s["table"], s["lens"], s["parents"], refs)
            short = ops.reserve_pages(table, lens, refs, data, tokens=1, cache_scales=scales)
        else:
            table, lens = plain_fork(s["table"], s["lens"], s["parents"], refs)
            short = plain_reserve(table, lens, refs, data, scales, 1)
        return (table, lens, refs, short) + _values(data, scales)
    table = s["table"].clone()
    if own:
        ops.free_pages(table, refs, s["lost"])
        page_map, live = ops.compact_pages(table, refs, data, cache_scales=scales)
    else:
        plain_free(table, refs, s["lost"])
        page_map, live = plain_compact(table, refs, data, scales)
    return (table, refs, page_map, live) + _values(data, scales)


# ------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    """log softmax and its entropy in 64 bits, 256 rows at a time; moving pages computes no numbers."""
    if case["op"] not in ("token_logprobs", "linear_logprobs"):
        return None
    s = prepare(case, seed)
    ids = s["ids"].view(case["rows"], -1).long()
    top_k = case.get("top_k", 0)
    weight = s["w"].double().t() if "w" in s else None
    out = []
    for r in range(0, case["rows"], 256):
        x = s["x"][r:r + 256].double() @ weight if weight is not None else s["logits"][r:r + 256].double()
        empty = (x == float("-inf")).all(1, keepdim=True)
        x = x - torch.where(empty, 0.0, x.amax(1, keepdim=True))  # first: a row may be all of its type's lowest value
        logp = x - torch.where(empty, 0.0, torch.log(x.exp().sum(1, keepdim=True)))
        entropy = -torch.where(logp == float("-inf"), 0.0, logp.exp() * logp).sum(1)
        i = ids[r:r + 256]
        given = torch.where(i < 0, 0.0, logp.gather(1, i.clamp(min=0)))
        best = torch.sort(logp, dim=1, descending=True, stable=True) if top_k else None
        value = best.values[:, :top_k] if top_k else logp[:, :0]
        index = torch.where(value == float("-inf"), -1, best.indices[:, :top_k]) if top_k else i[:, :0]
        out.append((given, entropy, value, index.int()))
    given, entropy, value, index = (torch.cat([o[j] for o in out]) for j in range(4))
    given = given.view(s["ids"].shape)
    return (given, entropy, value, index) if case["op"] == "token_logprobs" else (given, entropy)
