"""Sharing pages of a paged cache between rows: fork, reserve, free, compact and copy
against a model of them in plain Python."""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"


def _ops():
    from sparkpipe_rs_b200 import ops

    return ops


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


class Model:
    """The same operations one row after the other on lists; the cache as [planes][layers, slots, row] on the CPU."""

    def __init__(self, table, lens, refs, planes, bs):
        self.table = [list(r) for r in table]
        self.lens, self.refs, self.bs = list(lens), list(refs), bs
        self.planes = [p.clone() for p in planes]

    def held(self, e):
        return 0 <= e < len(self.refs)

    def fork(self, parents):
        cols = len(self.table[0]) if self.table else 0
        new, lens = [], []
        for p in parents:
            ok = 0 <= p < len(self.table)
            n = self.lens[p] if ok else 0
            used = -(-max(n, 0) // self.bs)
            new.append([self.table[p][c] if ok and c < used else -1 for c in range(cols)])
            lens.append(n)
        for r in self.table:
            for e in r:
                if self.held(e):
                    self.refs[e] -= 1
        for r in new:
            for e in r:
                if self.held(e):
                    self.refs[e] += 1
        self.table, self.lens = new, lens

    def copy_tokens(self, src, dst, n):
        for p in self.planes:
            p[:, dst * self.bs:dst * self.bs + n] = p[:, src * self.bs:src * self.bs + n]

    def reserve(self, tokens):
        free = [p for p, r in enumerate(self.refs) if r <= 0]
        start_refs = list(self.refs)
        left, at, short, tails, stuck = len(free), 0, [], [], []
        for b, row in enumerate(self.table):
            n = max(self.lens[b], 0)
            want = tokens[b] if isinstance(tokens, list) else (tokens if n > 0 else 0)
            col = n // self.bs
            private = False
            if want > 0 and n % self.bs and col < len(row) and self.held(row[col]):
                private = start_refs[row[col]] - tails.count(row[col]) > 1
                tails.append(row[col])
            first, last = -(-n // self.bs), -(-(n + want) // self.bs) if want > 0 else 0
            fresh = [c for c in range(first, min(last, len(row))) if row[c] < 0]
            need = private + len(fresh)
            ok = at + need <= left
            short.append(0 if ok else need)
            if need and not ok and col < len(row):
                stuck.append(row[col] if private else None)
            # the page that a row was to keep still has an unserved one on it
            if not need and want > 0 and n % self.bs and col < len(row) and row[col] >= 0 and row[col] in stuck:
                short[-1] = 1
            if ok and need:
                g = at
                if private:
                    old, page = row[col], free[g]
                    g += 1
                    self.copy_tokens(old, page, n % self.bs)
                    self.refs[old] -= 1
                    self.refs[page] = 1
                    row[col] = page
                for c in fresh:
                    row[c] = free[g]
                    self.refs[free[g]] = 1
                    g += 1
            at += need
        return short

    def free(self, rows):
        for b in set(rows):
            if 0 <= b < len(self.table):
                for c, e in enumerate(self.table[b]):
                    if self.held(e):
                        self.refs[e] -= 1
                    self.table[b][c] = -1

    def compact(self):
        live = [p for p, r in enumerate(self.refs) if r > 0]
        L = len(live)
        holes = [p for p in range(L) if self.refs[p] <= 0]
        moving = [p for p in live if p >= L]
        page_map = [p if r > 0 else -1 for p, r in enumerate(self.refs)]
        for p, h in zip(moving, holes):
            self.copy_tokens(p, h, self.bs)
            page_map[p] = h
            self.refs[h], self.refs[p] = self.refs[p], 0
        for row in self.table:
            for c, e in enumerate(row):
                if self.held(e):
                    row[c] = page_map[e]
        return page_map, L


CACHES = ["bf16", "fp8", "words", "view"]


def make_cache(kind, layers, pages, bs, seed):
    """(data, scales): bf16 rows of 576, the fp8 cache, rows of 5 words, or a layer-strided view of a wider cache."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    slots = pages * bs
    if kind == "words":
        return torch.randn(layers, slots, 5, device=DEV, generator=g), None
    if kind == "view":
        return torch.randn(layers, slots + 24, 24, device=DEV, generator=g).bfloat16()[:, :slots], None
    data = torch.randn(layers, slots, 576, device=DEV, generator=g).bfloat16()
    if kind == "bf16":
        return data, None
    return data.to(torch.float8_e4m3fn).view(torch.uint8), torch.rand(layers, slots, 5, device=DEV, generator=g)


def planes(data, scales):
    return [data] if scales is None else [data, scales]


def random_state(rng, rows, cols, pages, bs):
    """A consistent table: pages shared between some rows up to a common length, refs to match."""
    free = list(range(pages))
    rng.shuffle(free)
    table, lens = [], []
    for _ in range(rows):
        if table and rng.random() < 0.4:
            p = rng.randrange(len(table))
            table.append(list(table[p]))
            lens.append(lens[p])
            continue
        n = rng.choice([0, 0, 1, bs - 1, bs, bs + 1, rng.randrange(0, cols * bs + 1)])
        n = max(0, min(n, cols * bs, len(free) * bs))
        used = -(-n // bs)
        table.append([free.pop() for _ in range(used)] + [-1] * (cols - used))
        lens.append(n)
    refs = [0] * pages
    for r in table:
        for e in r:
            if e >= 0:
                refs[e] += 1
    return table, lens, refs


def same(model, table, refs, data, scales, what):
    assert table.cpu().tolist() == model.table, what
    assert refs.cpu().tolist() == model.refs, what
    for got, want in zip(planes(data, scales), model.planes):
        assert torch.equal(got.cpu(), want), what


@pytest.mark.parametrize("kind", CACHES)
@pytest.mark.parametrize("rows,cols,pages,bs,layers", [(1, 1, 1, 1, 1), (3, 4, 9, 4, 2), (8, 5, 40, 16, 3),
                                                       (33, 7, 150, 64, 2), (200, 3, 900, 3, 1), (5, 2, 4, 64, 27)])
def test_life_of_a_table(kind, rows, cols, pages, bs, layers):
    """Rounds of fork, reserve, tokens, free and compact; pages run out in some of them."""
    ops = _ops()
    rng = random.Random(rows * 7 + pages + len(kind))
    t, n, r = random_state(rng, rows, cols, pages, bs)
    data, scales = make_cache(kind, layers, pages, bs, rows)
    m = Model(t, n, r, [p.cpu() for p in planes(data, scales)], bs)
    table, lens, refs = ints(t).view(rows, cols), ints(n), ints(r)
    for step in range(4):
        parents = [rng.choice([-1, rows + 3] + list(range(rows)) * 3) for _ in range(rows)]
        table, lens = ops.fork_pages(table, lens, ints(parents), refs, block_size=bs)
        m.fork(parents)
        assert lens.cpu().tolist() == m.lens
        same(m, table, refs, data, scales, f"fork {step}")
        per_row = step % 2 == 1
        tokens = [rng.choice([0, -3, 1, 1, bs, 2 * bs + 1]) for _ in range(rows)] if per_row else 1
        short = ops.reserve_pages(table, lens, refs, data, ints(tokens) if per_row else tokens, block_size=bs,
                                  cache_scales=scales)
        assert short.cpu().tolist() == m.reserve(tokens)
        same(m, table, refs, data, scales, f"reserve {step}")
        for b in range(rows):  # the tokens that fit in the pages that a row has now
            room = sum(e >= 0 for e in m.table[b]) * bs
            m.lens[b] = min(room, max(m.lens[b], 0) + max(0, tokens[b] if per_row else int(m.lens[b] > 0)))
        lens = ints(m.lens)
        gone = [rng.randrange(-2, rows + 2) for _ in range(rows // 3)]
        gone += gone[:1]
        ops.free_pages(table, refs, ints(gone))
        m.free(gone)
        m.lens = [0 if b in gone else v for b, v in enumerate(m.lens)]
        lens = ints(m.lens)
        same(m, table, refs, data, scales, f"free {step}")
        page_map, live = ops.compact_pages(table, refs, data, block_size=bs, cache_scales=scales)
        want_map, want_live = m.compact()
        assert page_map.cpu().tolist() == want_map and int(live) == want_live
        same(m, table, refs, data, scales, f"compact {step}")
    ops.free_pages(table, refs)
    assert int(refs.abs().sum()) == 0 and int((table != -1).sum()) == 0
    assert ops.status_word() == 0


def test_shared_last_page():
    """Three rows and a holder outside the table share a partly filled page: every row gets a copy;
    without the outsider the last row keeps the page."""
    ops = _ops()
    for outside in (0, 1):
        data, scales = make_cache("fp8", 2, 10, 64, 4)
        table, lens, refs = ints([[3, -1], [3, -1], [3, -1]]), ints([7, 7, 7]), ints([0] * 10)
        refs[3] = 3 + outside
        before = data.clone()
        assert ops.reserve_pages(table, lens, refs, data, cache_scales=scales).tolist() == [0, 0, 0]
        assert table.tolist() == [[0, -1], [1, -1], [2 if outside else 3, -1]]
        assert refs.tolist()[:5] == ([1, 1, 1, 1, 0] if outside else [1, 1, 0, 1, 0])
        for p in (0, 1):
            assert torch.equal(data[:, p * 64:p * 64 + 7], before[:, 192:199])
            assert torch.equal(data[:, p * 64 + 7:p * 64 + 64], before[:, p * 64 + 7:p * 64 + 64])


def test_no_page_left_for_a_shared_one():
    """Two rows of different lengths on one page, one page too few: neither may write, and with
    a free page the first leaves with its tokens and the second keeps the page."""
    ops = _ops()
    for pages, short, table in ((1, [1, 1], [[0], [0]]), (2, [0, 0], [[1], [0]])):
        data, _ = make_cache("bf16", 1, pages, 16, 3)
        before = data.clone()
        t, refs = ints([[0], [0]]), ints([2, 0][:pages])
        assert ops.reserve_pages(t, ints([12, 5]), refs, data, 2, block_size=16).tolist() == short
        assert t.tolist() == table
        assert torch.equal(data[:, 16:28], before[:, :12]) if pages == 2 else torch.equal(data, before)


@pytest.mark.parametrize("pages", [8192, 20000])
def test_many_rows_and_pages(pages):
    """The most rows of one call, more pages than one sweep of the index kernels (and than their shared memory)."""
    ops = _ops()
    rows, bs = ops.kernels().PAGES_MAX_ROWS, 4
    rng = random.Random(5)
    t, n, r = random_state(rng, rows, 3, pages, bs)
    data = torch.randn(1, pages * bs, 2, device=DEV)
    m = Model(t, n, r, [data.cpu()], bs)
    table, lens, refs = ints(t), ints(n), ints(r)
    for tokens in (2, 17):  # the second asks for several pages a row, over four thousand in all
        if tokens == 17:
            table = torch.cat([table, torch.full((rows, 5), -1, dtype=torch.int32, device=DEV)], 1).contiguous()
            m.table = [row + [-1] * 5 for row in m.table]
        short = ops.reserve_pages(table, lens, refs, data, tokens, block_size=bs)
        assert short.cpu().tolist() == m.reserve(tokens)
        same(m, table, refs, data, None, "reserve")
    ops.free_pages(table, refs, ints(list(range(0, rows, 2))))
    m.free(list(range(0, rows, 2)))
    page_map, live = ops.compact_pages(table, refs, data, block_size=bs)
    assert page_map.cpu().tolist() == m.compact()[0]
    same(m, table, refs, data, None, "compact")


@pytest.mark.parametrize("kind", CACHES)
@pytest.mark.parametrize("bs", [1, 16, 64])
def test_copy_pages(kind, bs):
    ops = _ops()
    data, scales = make_cache(kind, 3, 40, bs, bs)
    want = [p.clone() for p in planes(data, scales)]
    src, dst = [5, 5, -1, 7, 9, 30, 12], [0, 39, 3, -1, 9, 31, 14]
    for a, b in zip(src, dst):
        if a >= 0 and b >= 0:
            for p in want:
                p[:, b * bs:(b + 1) * bs] = p[:, a * bs:(a + 1) * bs]
    ops.copy_pages(data, ints(src), ints(dst), block_size=bs, cache_scales=scales)
    for got, w in zip(planes(data, scales), want):
        assert torch.equal(got, w)
    n = ops.launch_count()
    ops.copy_pages(data, ints([]), ints([]), block_size=bs, cache_scales=scales)
    assert ops.launch_count() == n and ops.status_word() == 0


@pytest.mark.parametrize("src,dst", [([1, 2], [5, 5]), ([1, 2], [2, 3]), ([1, 4], [3, 1]), ([40], [2]), ([2], [40]),
                                     ([-2], [3])])
def test_copy_refused(src, dst):
    """Pairs whose order would matter, and pages outside the cache: nothing is copied, the status word is set."""
    ops = _ops()
    data, _ = make_cache("bf16", 2, 40, 4, 1)
    want = data.clone()
    ops.copy_pages(data, ints([9] + src), ints([20] + dst), block_size=4)
    assert torch.equal(data, want) and ops.status_word() == 5
    ops.clear_status()
    ops.copy_pages(data, ints([9]), ints([20]), block_size=4)
    want[:, 80:84] = want[:, 36:40]
    assert torch.equal(data, want) and ops.status_word() == 0


def test_offsets_past_32_bits():
    """A plane of more than 2^32 bytes per layer, and layers past 2^33."""
    ops = _ops()
    pages = 62000
    data = torch.zeros(2, pages * 64, 576, dtype=torch.bfloat16, device=DEV)
    data[1, -64:] = torch.randn(64, 576, device=DEV).bfloat16()
    data[0, -64:] = 2.0
    ops.copy_pages(data, ints([pages - 1]), ints([pages - 2]))
    assert torch.equal(data[:, -128:-64], data[:, -64:])
    refs = torch.zeros(pages, dtype=torch.int32, device=DEV)
    refs[-1] = 1
    table = ints([[pages - 1]])
    page_map, live = ops.compact_pages(table, refs, data)
    assert table.tolist() == [[0]] and int(live) == 1 and int(page_map[-1]) == 0
    assert torch.equal(data[:, :64], data[:, -64:]) and int(refs[0]) == 1 and int(refs.sum()) == 1


def test_captured_beam_steps():
    """Fork and reserve captured once and replayed with new parents on the same tables."""
    ops = _ops()
    rows, cols, pages, bs = 6, 4, 60, 8
    rng = random.Random(2)
    t, n, r = random_state(rng, rows, cols, pages, bs)
    data, _ = make_cache("bf16", 2, pages, bs, 7)
    m = Model(t, n, r, [data.cpu()], bs)
    table, lens, refs, parents = ints(t), ints(n), ints(r), ints([0] * rows)

    def step():
        new, new_lens = ops.fork_pages(table, lens, parents, refs, block_size=bs)
        short = ops.reserve_pages(new, new_lens, refs, data, 1, block_size=bs)
        table.copy_(new)
        lens.copy_(new_lens)
        lens.add_((lens > 0).int())
        return short

    g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s), torch.cuda.graph(g, stream=s):
        short = step()
    torch.cuda.current_stream().wait_stream(s)
    for _ in range(12):
        p = [rng.randrange(rows) for _ in range(rows)]
        parents.copy_(ints(p))
        g.replay()
        m.fork(p)
        want = m.reserve(1)
        m.lens = [v + int(v > 0) for v in m.lens]
        assert short.cpu().tolist() == want
        assert lens.cpu().tolist() == m.lens
        same(m, table, refs, data, None, "replay")


@pytest.mark.parametrize("pages", [8192, 8193, 20000])
def test_no_page_left_in_a_large_cache(pages):
    """Pages run out among 1,000 rows that share last pages, with the counts in shared memory and read from
    refs: what a row lacks goes by the counts before the call, not by what other rows changed meanwhile."""
    ops = _ops()
    rows, bs = 1000, 4
    rng = random.Random(pages)
    shared = rng.sample(range(pages), 250)  # four rows to a page, of one to three tokens
    t = [[p] for p in shared for _ in range(4)]
    n = [rng.randrange(1, bs) for _ in range(rows)]
    r = [1] * pages
    for p in shared:
        r[p] = 4
    for p in rng.sample([p for p in range(pages) if p not in set(shared)], 400):  # 400 pages for 750 rows that leave
        r[p] = 0
    for _ in range(5):
        data = torch.randn(1, pages * bs, 2, device=DEV)
        m = Model(t, n, r, [data.cpu()], bs)
        table, lens, refs = ints(t), ints(n), ints(r)
        short = ops.reserve_pages(table, lens, refs, data, 1, block_size=bs)
        want = m.reserve(1)
        assert sum(want) > 0 and short.cpu().tolist() == want
        same(m, table, refs, data, None, pages)


class CheckedModel(Model):
    """Reserves like Model, but leaves rows alone whose partly filled last page is missing, and with `strict`
    those whose tokens go past the table's width."""

    def reserve(self, tokens, strict=False):
        want = list(tokens) if isinstance(tokens, list) else [tokens if n > 0 else 0 for n in self.lens]
        lacks = [0] * len(self.table)
        for b, row in enumerate(self.table):
            n = max(self.lens[b], 0)
            if want[b] <= 0:
                continue
            first, end = -(-n // self.bs), -(-(n + want[b]) // self.bs)
            lost = n % self.bs and n // self.bs < len(row) and not self.held(row[n // self.bs])
            past = max(0, end - len(row)) if strict else 0
            if lost or past:
                lacks[b] = bool(lost) + past + sum(e < 0 for e in row[first:end])
                want[b] = 0
        return [a + b for a, b in zip(super().reserve(want), lacks)]


def test_no_room_in_the_table():
    """Rows whose tokens go past the table's width: with `strict` each gets nothing and lacks what it would need,
    the rows around them are served, and one that shares a page with such a row leaves it."""
    ops = _ops()
    bs, pages = 4, 12
    t = [[0, 1], [2, 3], [4, 5], [6, -1], [7, 5]]
    n, tokens = [8, 7, 6, 4, 5], [1, 2, 2, 9, 1]  # full; straddling; fits (shared page); fits in no table; fits
    n[1], t[1] = 6, [2, 5]
    tokens[1] = 5                                  # holds page 5 as well, and goes past the width
    r = [0] * pages
    for row in t:
        for e in row:
            if e >= 0:
                r[e] += 1
    data = torch.randn(2, pages * bs, 2, device=DEV)
    m = CheckedModel(t, n, r, [data.cpu()], bs)
    table, lens, refs = ints(t), ints(n), ints(r)
    short = ops.reserve_pages(table, lens, refs, data, ints(tokens), block_size=bs, strict=True)
    assert short.tolist() == [1, 1, 0, 3, 0]
    assert table.tolist() == [[0, 1], [2, 5], [4, 3], [6, -1], [7, 8]] and refs.tolist()[5] == 1
    assert m.reserve(tokens, True) == short.tolist()
    same(m, table, refs, data, None, "strict")
    one = ops.reserve_pages(ints([[0, 1]]), ints([2**31 - 1]), refs, data, 2**31 - 1, block_size=1, strict=True)
    assert int(one) == 2**30 - 1  # 2^32 - 4 pages past the width, as many as are counted
    # without it the width bounds a row
    assert ops.reserve_pages(ints([[0, 1]]), ints([8]), ints(r), data, 1, block_size=bs).tolist() == [0]


def test_last_page_missing():
    """A row of some tokens whose last page is not there, or is no page of the cache, may not be written."""
    ops = _ops()
    bs = 4
    t, n = [[0, -1, -1], [1, 99, -1], [2, 3, -1], [-1, -1, -1]], [6, 5, 7, 0]
    r = [1, 1, 1, 1, 0, 0, 0, 0, 0]
    for tokens, lacks in ((1, [1, 1, 0, 0]), (5, [2, 2, 0, 0])):
        data = torch.randn(1, 9 * bs, 2, device=DEV)
        m = CheckedModel(t, n, r, [data.cpu()], bs)
        table, refs = ints(t), ints(r)
        short = ops.reserve_pages(table, ints(n), refs, data, tokens, block_size=bs)
        assert short.tolist() == lacks == m.reserve(tokens)
        same(m, table, refs, data, None, tokens)


@pytest.mark.parametrize("kind", ["bf16", "fp8"])
@pytest.mark.parametrize("rows,cols,pages,bs,layers", [(1, 1, 3, 1, 1), (5, 2, 9, 4, 2), (33, 3, 90, 16, 2),
                                                       (200, 3, 9000, 3, 1)])
def test_strict_rounds(kind, rows, cols, pages, bs, layers):
    """Tables too narrow for many of their rows, pages that run out in some rounds, lengths past the width."""
    ops = _ops()
    rng = random.Random(rows + pages)
    for _ in range(6):
        t, n, r = random_state(rng, rows, cols, pages, bs)
        for b in range(0, rows, 9):  # a last page that is lost, a length that the table does not hold
            c = n[b] // bs
            if n[b] % bs and c < cols and rng.random() < 0.5:
                r[t[b][c]] -= 1
                t[b][c] = -1
            elif rng.random() < 0.3:
                n[b] = cols * bs + rng.randrange(3 * bs)
        data, scales = make_cache(kind, layers, pages, bs, rows)
        m = CheckedModel(t, n, r, [p.cpu() for p in planes(data, scales)], bs)
        tokens = [rng.choice([0, -1, 1, 1, bs, 2 * bs + 1]) for _ in range(rows)]
        table, refs = ints(t).view(rows, cols), ints(r)
        short = ops.reserve_pages(table, ints(n), refs, data, ints(tokens), block_size=bs, cache_scales=scales, strict=True)
        assert short.cpu().tolist() == m.reserve(tokens, True)
        same(m, table, refs, data, scales, "strict")
    assert ops.status_word() == 0
