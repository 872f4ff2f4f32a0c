"""Forks, compaction and copies of a cache's pages: against the definition row by row, and by what a program needs of them
(every sequence finds its tokens, nobody's last page is another's, uses add up).  All results are exact."""

import random

import pytest
import torch

from tttj_2026_amd import ops

pytestmark = pytest.mark.gpu

E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _held(n, page, columns):
    return min(-(-max(n, 0) // page), columns)


def _fork(table, lengths, uses, parents, counts, page):
    """The definition: (table, lengths, uses, copies (source, target, tokens))."""
    batch, columns, pages = len(table), len(table[0]) if table else 0, len(uses)
    uses, most = list(uses), columns * page
    rows = []
    for b in range(batch):
        p = parents[b]
        if 0 <= p < batch:
            before = min(max(lengths[p], 0), most)
            after = min(max(before + counts[b], 0), most)
            rows.append((p, after, min(before, after)))
        else:
            rows.append((None, 0, 0))
    for b in range(batch):
        for i in range(_held(lengths[b], page, columns)):
            if 0 <= table[b][i] < pages:
                uses[table[b][i]] -= 1
    first = {}
    for b, (p, after, kept) in enumerate(rows):
        for i in range(kept // page):
            if 0 <= table[p][i] < pages:
                uses[table[p][i]] += 1
        if kept % page:
            first.setdefault(table[p][kept // page], b)
    held_whole = list(uses)
    out, copies = [], []
    for b, (p, after, kept) in enumerate(rows):
        mine = list(table[p][:_held(kept, page, columns)]) if p is not None else []
        copy = None
        if kept % page and 0 <= mine[-1] < pages:
            if first[mine[-1]] == b and held_whole[mine[-1]] == 0:
                uses[mine[-1]] += 1
            else:
                copy = mine.pop()
        out.append((mine, after, copy, kept % page))
    free = [i for i, n in enumerate(uses) if n == 0]
    new = []
    for mine, after, copy, part in out:
        for i in range(len(mine), _held(after, page, columns)):
            mine.append(free.pop(0) if free else -1)
            if mine[-1] >= 0:
                uses[mine[-1]] = 1
            if copy is not None:
                copies.append((copy, mine[-1], part))
                copy = None
        new.append(mine + [-1] * (columns - len(mine)))
    return new, [r[1] for r in rows], uses, copies


def _world(rng, batch, columns, page, pages, share=True):
    """A state as calls leave it: (table, lengths, uses)."""
    order = list(range(pages))
    rng.shuffle(order)
    uses, table, lengths = [0] * pages, [], []
    for b in range(batch):
        length = rng.choice([0, 1, page, columns * page, rng.randint(0, columns * page), rng.randint(0, 2 * page)])
        length = min(length, columns * page)
        mine = []
        if share and b and rng.random() < 0.6:  # whole pages of an earlier one
            other = rng.randrange(b)
            n = rng.randint(0, min(lengths[other], length) // page)
            mine = table[other][:n]
        need = _held(length, page, columns)
        if len(mine) + len(order) < need:
            length = len(mine) * page
            need = len(mine)
        while len(mine) < need:
            mine.append(order.pop())
        for p in mine:
            uses[p] += 1
        lengths.append(length)
        # what lies behind counts for nothing
        table.append(mine + [rng.choice([-1, pages, rng.randrange(pages), 1 << 30]) for _ in range(columns - len(mine))])
    for p in rng.sample(range(pages), min(3, pages)):  # kept prompts
        uses[p] += 1 if uses[p] else 0
    return table, lengths, uses


def _caches(pages, page, seed=0, layers=2, heads=3, hd=16):
    """K and V of layers in 16 bits, one layer in 8 bits with its scales, and a tensor in another order."""
    g = torch.Generator().manual_seed(seed)
    kv = torch.randn(layers, 2, pages, page, heads, hd, generator=g).half().cuda()
    both = torch.randn(pages, 2, page, heads, hd, generator=g).bfloat16().cuda()  # a page's halves side by side
    eight = torch.randint(0, 127, (2, pages, page, heads, hd), generator=g, dtype=torch.uint8).cuda().view(E4M3)
    scales = torch.randint(0, 255, (2, pages, page // 16, heads), generator=g, dtype=torch.uint8).cuda().view(E8M0)
    turned = torch.randn(pages, heads, page, 5, generator=g).cuda().transpose(1, 2)
    return [*kv.flatten(0, 1), *both.unbind(1), *eight, *scales, turned]


def _raw(t):
    return t.view(torch.uint8) if t.element_size() == 1 else t


def _copied(caches, copies, page):
    """The caches after the copies, by the definition."""
    out = [_raw(t).cpu().clone() for t in caches]
    for t, c in zip(caches, out):
        dense = t.is_contiguous() or t[0].is_contiguous()
        for source, target, tokens in copies:
            if target < 0:
                continue
            rows = -(-tokens * c.shape[1] // page) if dense else c.shape[1]
            c[target, :rows] = c[source, :rows]
    return out


def _equal(caches, want):
    for i, (t, c) in enumerate(zip(caches, want)):
        assert torch.equal(_raw(t).cpu(), c), i


@pytest.mark.parametrize("seed", range(60))
def test_fork(seed):
    rng = random.Random(seed)
    batch, columns, page = rng.choice([1, 2, 5, 16, 70]), rng.choice([1, 2, 5, 9]), rng.choice([16, 16, 32, 64])
    pages = rng.choice([batch * columns + 5, batch * columns // 2 + 2, 2 * batch * columns + 1])
    table, lengths, uses = _world(rng, batch, columns, page, pages)
    kind = seed % 4
    parents = [b if kind == 0 else rng.choice([-1, b, rng.randrange(batch), rng.randrange(batch), batch, 0])
               for b in range(batch)]
    counts = [rng.choice([0, 1, 1, 3, page, -1, -page, -5, rng.randint(-columns * page, columns * page),
                          2 ** 31 - 1, -2 ** 31]) for _ in range(batch)]
    if kind == 3:
        counts = [0] * batch
    caches = _caches(pages, page, seed)
    t, n, u = _i32(table), _i32(lengths), _i32(uses)
    new = _fork(table, lengths, uses, parents, counts, page)
    want = _copied(caches, new[3], page)
    before = [_raw(c).clone() for c in caches]
    got = ops.cache_fork(caches, t, n, u, None if kind == 0 else _i32(parents), None if kind == 3 else _i32(counts))
    for a, b in zip(got, new):
        assert a.tolist() == b
    _equal(caches, want)
    assert t.tolist() == table and n.tolist() == lengths and u.tolist() == uses
    # what a program needs: every row finds its tokens, and nobody else the page that it is about to write
    table2, lengths2, uses2 = (x.tolist() for x in got)
    for b, p in enumerate(parents):
        if not 0 <= p < batch:
            assert lengths2[b] == 0
            continue
        for i in range(0, min(lengths[p], lengths2[b]), page):
            rows = min(page, min(lengths[p], lengths2[b]) - i)
            old, now = table[p][i // page], table2[b][i // page]
            if now >= 0:
                for c, x in zip(caches, before):
                    part = -(-rows * c.shape[1] // page)
                    assert torch.equal(_raw(c)[now, :part], x[old, :part])
    counted = [0] * pages
    for r, n in zip(table2, lengths2):
        for p in r[:_held(n, page, columns)]:
            if p >= 0:
                counted[p] += 1
    holds = [a - b for a, b in zip(uses2, counted)]
    assert holds == [a - sum(p in r[:_held(n, page, columns)] for r, n in zip(table, lengths)) for p, a in enumerate(uses)]
    lasts = [r[min(lengths[q], n) // page] for r, n, q in zip(table2, lengths2, parents)
             if 0 <= q < batch and min(lengths[q], n) % page]
    lasts = [p for p in lasts if p >= 0]
    assert len(lasts) == len(set(lasts)) and all(uses2[p] == 1 for p in lasts)


@pytest.mark.parametrize("batch,columns,pages", [(3, 5, 4000), (1100, 2, 2500), (1, 5000, 6000), (2049, 3, 6000),
                                                 (70, 6, 16384), (70, 6, 16385), (40, 900, 50001)])
def test_fork_of_many(batch, columns, pages):
    """More rows, columns or pages than the block has threads, or LDS room for counters."""
    rng = random.Random(batch)
    table, lengths, uses = _world(rng, batch, columns, 16, pages)
    parents = [rng.choice([b, b, rng.randrange(batch), -1]) for b in range(batch)]
    counts = [rng.choice([0, 1, 20, -7]) for _ in range(batch)]
    caches = _caches(pages, 16)[-4::2] + _caches(pages, 16, 1)[-1:]
    new = _fork(table, lengths, uses, parents, counts, 16)
    want = _copied(caches, new[3], 16)
    got = ops.cache_fork(caches, _i32(table), _i32(lengths), _i32(uses), _i32(parents), _i32(counts))
    for a, b in zip(got, new):
        assert a.tolist() == b
    _equal(caches, want)
    table, lengths, uses = (x.tolist() for x in got)
    new = _compact(table, lengths, uses, 16)
    want = _copied(caches, new[2], 16)
    moved = ops.cache_compact(caches, *got)
    for a, b in zip(moved, new):
        assert a.tolist() == b
    _equal(caches, want)


def _compact(table, lengths, uses, page):
    total = sum(u > 0 for u in uses)
    moves = dict(zip([p for p, u in enumerate(uses) if u > 0 and p >= total],
                     [p for p, u in enumerate(uses) if u <= 0 and p < total]))
    uses = [u if p < total and u > 0 else 0 for p, u in enumerate(uses)], uses
    for p, q in moves.items():
        uses[0][q] = uses[1][p]
    columns = len(table[0])
    new = [[moves.get(p, p) if i < _held(n, page, columns) else -1 for i, p in enumerate(r)] for r, n in zip(table, lengths)]
    return new, uses[0], [(p, q, page) for p, q in moves.items()]


@pytest.mark.parametrize("seed", range(36))
def test_large_states(seed):
    """Either side of what one block does: 512 rows of 64 columns, 16384 pages."""
    rng = random.Random(seed)
    batch, columns, pages = [(512, 3, 900), (513, 3, 900), (8, 4096, 16384), (8, 4097, 16384), (257, 65, 9000), (513, 1, 2),
                             (513, 64, 16384), (5, 2, 16384), (5, 2, 16385), (1, 1, 20001), (0, 4, 16385), (2, 70, 40960),
                             ][seed % 12]
    table, lengths, uses = _world(rng, batch, columns, 16, pages)
    if seed // 12 == 1:  # the program holds most other pages, so that free ones run out
        uses = [u or (rng.random() < 0.97) * rng.randint(1, 3) for u in uses]
    elif seed // 12 == 2:  # or all
        uses = [u or 1 for u in uses]
    parents = [rng.choice([b, b, rng.randrange(batch), -1, batch, 0]) for b in range(batch)]
    counts = [rng.choice([0, 1, 20, -7, -1000, 16 * columns, 2 ** 31 - 1, -2 ** 31]) for _ in range(batch)]
    caches = _caches(pages, 16, heads=1)[-4::2]
    state = (_i32(table).view(batch, columns), _i32(lengths), _i32(uses))
    new = _fork(table, lengths, uses, parents, counts, 16) if batch else (table, lengths, uses, [])
    want = _copied(caches, new[3], 16)
    got = ops.cache_fork(caches, *state, _i32(parents), _i32(counts))
    for a, b in zip(got, new):
        assert a.tolist() == b
    _equal(caches, want)
    for state in (state, got):
        table, lengths, uses = (x.tolist() for x in state)
        new = _compact(table, lengths, uses, 16) if batch else _compact([[0]], [0], uses, 16)
        want = _copied(caches, new[2], 16)
        moved = ops.cache_compact(caches, *state)
        assert moved[0].tolist() == (new[0] if batch else [])
        assert moved[1].tolist() == new[1]
        _equal(caches, want)


def test_large_states_in_a_graph():
    """A fork and a compaction whose phases are launches, replayed over states that change."""
    batch, columns, pages = 40, 12, 17000
    caches, worlds = _caches(pages, 16, heads=1)[-5:-1:2], []
    rng = random.Random(1)
    for _ in range(3):
        state = _world(rng, batch, columns, 16, pages)
        worlds.append((*state, [rng.randrange(-1, batch) for _ in range(batch)], [rng.randint(-40, 40) for _ in range(batch)]))
    inputs = [_i32(x) for x in worlds[0]]

    def steps():
        table, lengths, uses = ops.cache_fork(caches, *inputs)
        return (lengths, *ops.cache_compact(caches, table, lengths, uses))

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        steps()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = steps()
    for table, lengths, uses, parents, counts in worlds + worlds[:1]:
        for x, y in zip(inputs, (table, lengths, uses, parents, counts)):
            x.copy_(_i32(y))
        forked = _fork(table, lengths, uses, parents, counts, 16)
        new = _compact(*forked[:3], 16)
        want = _copied(_copied(caches, forked[3], 16), new[2], 16)
        graph.replay()
        torch.cuda.synchronize()
        assert [x.tolist() for x in out] == [forked[1], new[0], new[1]]
        _equal(caches, want)
        torch.zeros(1000, device="cuda").sum().item()  # the program's own work between


@pytest.mark.parametrize("seed", range(24))
def test_compact(seed):
    rng = random.Random(seed)
    batch, columns, page = rng.choice([1, 2, 16, 70]), rng.choice([1, 2, 9]), rng.choice([16, 32])
    pages = rng.choice([1, 2, 3, batch * columns + 5, 4 * batch * columns + 1, 3000])
    table, lengths, uses = _world(rng, batch, columns, page, pages)
    caches = _caches(pages, page, seed)
    new = _compact(table, lengths, uses, page)
    want = _copied(caches, new[2], page)
    got = ops.cache_compact(caches, _i32(table), _i32(lengths), _i32(uses))
    for a, b in zip(got, new):
        assert a.tolist() == b
    used = sum(u > 0 for u in uses)
    assert all(u > 0 for u in got[1].tolist()[:used]) and not any(got[1].tolist()[used:])
    _equal(caches, want)


def test_copy():
    caches = _caches(50, 32)
    source, target = [3, 7, -1, 5, 50, 11, 12, 4], [20, 21, 22, 23, 24, 49, 1 << 30, 4]
    pairs = [(s, t, 32) for s, t in zip(source, target) if 0 <= s < 50 and 0 <= t < 50]
    want = _copied(caches, pairs, 32)
    ops.cache_copy(caches, _i32(source), _i32(target))
    _equal(caches, want)
    ops.cache_copy(caches, _i32([]), _i32([]))
    ops.cache_copy([caches[0]], _i32([0] * 1), _i32([1]))
    assert torch.equal(caches[0][1], caches[0][0])


@pytest.mark.parametrize("heads,hd,dtype", [(1, 1, torch.uint8), (3, 7, torch.uint8), (1, 3, torch.float16),
                                            (8, 256, torch.float16), (5, 80, torch.float32)])
def test_pages_of_any_size(heads, hd, dtype):
    """Odd numbers of bytes, pages that are not aligned, and pages of several pieces."""
    for offset in (0, 1, 2):
        flat = torch.randint(0, 100, (37 * 64 * heads * hd + offset,)).to(dtype).cuda()[offset:]
        t = flat.view(37, 64, heads, hd)
        want = t.cpu().clone()
        table, lengths, uses = [[4, 9, -1], [-1] * 3], [64 + 37, 0], [0] * 37
        uses[4] = uses[9] = 1
        got = ops.cache_fork([t], _i32(table), _i32(lengths), _i32(uses), _i32([0, 0]))
        want[0, :37] = want[9, :37]
        assert got[0].tolist() == [[4, 9, -1], [4, 0, -1]]
        assert torch.equal(t.cpu(), want)
        ops.cache_copy([t], _i32([36, 2]), _i32([1, 3]))
        want[1], want[3] = want[36], want[2]
        assert torch.equal(t.cpu(), want)


def test_many_tensors():
    """More tensors than one launch takes."""
    kv = torch.randn(70, 9, 16, 2, 8).half().cuda()
    want = kv.cpu().clone()
    ops.cache_copy(list(kv), _i32([1, 5]), _i32([8, 2]))
    want[:, 8], want[:, 2] = want[:, 1], want[:, 5]
    assert torch.equal(kv.cpu(), want)


def test_offsets_past_32_bits():
    t = torch.zeros(70, 256, 64, 1024, dtype=torch.float16, device="cuda")  # pages of 32 MiB
    t[1, :100], t[69] = 3.0, 5.0
    t[1, 99, 63, 1023] = 7.0
    got = ops.cache_fork([t], _i32([[1, -1], [1, -1]]), _i32([100, 0]), _i32([1] * 2 + [2] * 66 + [0, 1]), _i32([0, 0]))
    assert got[0].tolist() == [[1, -1], [68, -1]]
    assert bool((t[68, :100] == t[1, :100]).all()) and not bool(t[68, 100:].any())
    ops.cache_copy([t], _i32([69]), _i32([67]))
    assert bool((t[67] == 5).all())


def test_nothing_to_do():
    caches = _caches(7, 16)
    before = [_raw(c).clone() for c in caches]
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    uses = _i32([1, 0, 0, 2, 0, 0, 0])
    table, lengths, held = ops.cache_fork(caches, none.view(0, 1), none, uses, none, none)
    assert table.shape == (0, 1) and lengths.shape == (0,) and torch.equal(held, uses)
    for c, x in zip(caches, before):
        assert torch.equal(_raw(c), x)
    table, held = ops.cache_compact(caches, none.view(0, 1), none, uses)
    assert held.tolist() == [1, 2, 0, 0, 0, 0, 0]


def test_strides_of_the_state():
    """Columns of a wider table, and a transposed one."""
    rng = random.Random(5)
    table, lengths, uses = _world(rng, 6, 4, 16, 40)
    parents, counts = [0, 0, 1, 5, -1, 2], [1] * 6
    new = _fork(table, lengths, uses, parents, counts, 16)
    wide = torch.full((6, 9), 3, dtype=torch.int32, device="cuda")
    wide[:, 2:6] = _i32(table)
    for t in (wide[:, 2:6], _i32(table).T.contiguous().T):
        got = ops.cache_fork(_caches(40, 16), t, _i32(lengths), _i32(uses), _i32(parents), _i32(counts))
        for a, b in zip(got, new):
            assert a.tolist() == b


def test_graphs_and_streams():
    """A step of a program in a graph: state in, state out, copied back and replayed."""
    rng = random.Random(9)
    table, lengths, uses = _world(rng, 12, 6, 16, 120)
    parents, counts = [0, 0, 1, 2, 2, 2, 6, 7, -1, 9, 10, 11], [1] * 12
    caches = _caches(120, 16, 3)
    want = [c.clone() for c in caches]
    state = [_i32(table), _i32(lengths), _i32(uses)]
    eager = [s.clone() for s in state]
    p, c = _i32(parents), _i32(counts)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.cache_fork([x.clone() for x in caches], *state, p, c)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for s, x in zip(state, ops.cache_fork(caches, *state, p, c)):
            s.copy_(x)
    for step in range(5):
        graph.replay()
        torch.cuda.synchronize()
        eager = list(ops.cache_fork(want, *eager, p, c))
        torch.cuda.synchronize()
        for s, x in zip(state, eager):
            assert torch.equal(s, x), step
        for a, b in zip(caches, want):
            assert torch.equal(_raw(a), _raw(b)), step
