"""The pages of a KV cache: reserve, fork, free, compact and copy against plain lists; whole numbers, so all exact."""
import random

import pytest
import torch

from tests import paged_reference as ref
from vibe_compiler_b200.backend import WB200Error
from vibe_compiler_b200.paged_cache import PageTables, PagedCache

pytestmark = pytest.mark.gpu


def state(sequences, width, pages, size, seed, fill=0.6, pad=0):
    """Sequences of random lengths on random pages; the table is a view with `pad` columns more behind its rows."""
    rng = random.Random(seed)
    table = torch.full((sequences, width + pad), -1, dtype=torch.int32)
    lengths, refs = torch.zeros(sequences, dtype=torch.int32), torch.zeros(pages, dtype=torch.int32)
    free = list(range(pages))
    rng.shuffle(free)
    budget = int(pages * fill)
    for s in range(sequences):
        if rng.random() < 0.25:
            continue
        tokens = rng.randint(1, width * size)
        need = -(-tokens // size)
        if need > budget:
            continue
        budget -= need
        lengths[s] = tokens
        for j in range(need):
            table[s, j] = free.pop()
            refs[table[s, j]] = 1
    return table.cuda()[:, :width], lengths.cuda(), refs.cuda()


def agree(plain, table, lengths, refs):
    assert table.tolist() == plain.table and lengths.tolist() == plain.lengths and refs.tolist() == plain.refs


SIZES = [(1, 1, 1, 1), (5, 3, 9, 4), (33, 17, 200, 16), (300, 40, 7001, 3), (64, 700, 20000, 16)]


@pytest.mark.parametrize("sequences,width,pages,size", SIZES)
@pytest.mark.parametrize("in_place", [False, True])
def test_reserve_takes_the_lowest_free_pages_in_order(backend, sequences, width, pages, size, in_place):
    for seed in range(3):
        table, lengths, refs = state(sequences, width, pages, size, seed, pad=seed)
        rng = random.Random(seed)
        more = [rng.choice((-5, 0, 1, 1, 1, size, 3 * size)) for _ in range(sequences)]
        wanted = torch.tensor([min(n + m, width * size) for n, m in zip(lengths.tolist(), more)], dtype=torch.int32).cuda()
        plain = ref.Pages(table, lengths, refs, size)
        before = table.clone(), lengths.clone(), refs.clone()
        out = (table, lengths, refs) if in_place else None
        got = backend.pages_reserve(table, lengths, refs, wanted, size, out=out)
        assert plain.reserve(wanted) == int(got[3])
        agree(plain, *got[:3])
        if not in_place:
            assert all(torch.equal(a, b) for a, b in zip((table, lengths, refs), before))
    backend.poll()


def test_reserve_changes_nothing_when_it_cannot(backend):
    table, lengths, refs = state(20, 10, 120, 8, 1, fill=0.9)
    free = int((refs == 0).sum())
    empty = int((lengths == 0).nonzero()[0])
    for wanted_pages, outcome in ((free, 0), (free + 3, 3)):
        wanted = torch.zeros_like(lengths)
        spread = wanted_pages
        for s in (lengths == 0).nonzero().flatten().tolist():
            wanted[s] = min(spread, 10) * 8
            spread -= min(spread, 10)
        if spread:
            continue
        got = backend.pages_reserve(table, lengths, refs, wanted, 8)
        assert int(got[3]) == outcome
        if outcome:
            assert torch.equal(got[0], table) and torch.equal(got[1], lengths) and torch.equal(got[2], refs)
    wanted = torch.zeros_like(lengths)
    wanted[empty] = 81
    got = backend.pages_reserve(table, lengths, refs, wanted, 8)
    assert int(got[3]) == -1 and torch.equal(got[0], table) and torch.equal(got[1], lengths) and torch.equal(got[2], refs)
    backend.poll()


@pytest.mark.parametrize("sequences,width,pages,size", SIZES[1:])
@pytest.mark.parametrize("in_place", [False, True])
def test_fork_then_free_then_compact(backend, sequences, width, pages, size, in_place):
    for seed in range(3):
        table, lengths, refs = state(sequences, width, pages, size, 10 + seed, fill=0.5, pad=seed)
        plain = ref.Pages(table, lengths, refs, size)
        empty = (lengths == 0).nonzero().flatten().tolist()
        alive = (lengths > 0).nonzero().flatten().tolist()
        rng = random.Random(seed)
        children = rng.sample(empty, min(len(empty), 1 + seed * 7))
        parents = [rng.choice(alive) for _ in children]
        parents_t, children_t = torch.tensor(parents, dtype=torch.int32).cuda(), torch.tensor(children, dtype=torch.int32).cuda()
        out = (table, lengths, refs) if in_place else None
        table, lengths, refs, sources, destinations, result = backend.pages_fork(table, lengths, refs, parents_t, children_t, size, out=out)
        outcome = plain.fork(parents_t, children_t)
        assert (int(result), sources.tolist(), destinations.tolist()) == outcome
        agree(plain, table, lengths, refs)
        gone = rng.sample(alive, len(alive) // 2) + children[:1]
        gone_t = torch.tensor(gone + gone[:2] + [-1], dtype=torch.int32).cuda()     # some twice, one to pass over
        out = (table, lengths, refs) if in_place else None
        table, lengths, refs = backend.pages_free(table, lengths, refs, gone_t, size, out=out)
        plain.free(gone_t)
        agree(plain, table, lengths, refs)
        out = (table, refs) if in_place else None
        table, refs, sources, destinations = backend.pages_compact(table, lengths, refs, size, out=out)
        assert (sources.tolist(), destinations.tolist()) == plain.compact()
        agree(plain, table, lengths, refs)
    backend.poll()


def test_fork_refuses_what_is_no_fork(backend):
    table, lengths, refs = state(12, 6, 100, 8, 3, fill=0.5)
    lengths[0], lengths[1] = 0, 0
    alive = (lengths > 0).nonzero().flatten().tolist()
    a, b = alive[0], alive[1]
    for parents, children in (([a], [b]), ([a, b], [0, 0]), ([a], [12]), ([-1], [0]), ([a, 0], [0, 1])):
        p, c = torch.tensor(parents, dtype=torch.int32).cuda(), torch.tensor(children, dtype=torch.int32).cuda()
        got = backend.pages_fork(table, lengths, refs, p, c, 8)
        assert int(got[5]) == -1 and got[3].tolist() == [-1] * len(parents) == got[4].tolist()
        assert torch.equal(got[0], table) and torch.equal(got[1], lengths) and torch.equal(got[2], refs)
    full = torch.ones_like(refs)
    lengths[a] = lengths[a] // 8 * 8 + 5
    p, c = torch.tensor([a], dtype=torch.int32).cuda(), torch.tensor([0], dtype=torch.int32).cuda()
    assert int(backend.pages_fork(table, lengths, full, p, c, 8)[5]) == 1
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    got = backend.pages_fork(table, lengths, refs, none, none, 8)
    assert int(got[5]) == 0 and torch.equal(got[0], table)
    backend.poll()


def test_device_data_outside_the_arrays_is_reported(backend):
    table, lengths, refs = state(12, 6, 100, 8, 3, fill=0.5)
    alive = (lengths > 0).nonzero().flatten().tolist()
    for fault in ("sequence", "page", "length", "twice"):
        t, n, r = table.clone(), lengths.clone(), refs.clone()
        listed = torch.tensor([alive[0]], dtype=torch.int32).cuda()
        if fault == "sequence":
            listed[0] = 12
        elif fault == "page":
            t[alive[0], 0] = 100
        elif fault == "length":
            n[alive[0]] = 49
        else:
            r[t[alive[0], 0].long()] = 0
        backend.pages_free(t, n, r, listed, 8)
        with pytest.raises(WB200Error):
            backend.poll()
    backend.poll()
    n = lengths.clone()
    n[alive[0]] = -3
    assert int(backend.pages_reserve(table, n, refs, lengths, 8)[3]) == -1
    with pytest.raises(WB200Error):
        backend.poll()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("layout", ["rows", "heads", "pairs", "wide rows"])
@pytest.mark.parametrize("size,heads,head_dim", [(16, 8, 128), (5, 3, 36), (1, 1, 7), (64, 1, 64), (128, 8, 128)])
def test_copy_moves_whole_pages(backend, dtype, layout, size, heads, head_dim):
    pages, layers = 23, 3
    caches = []
    for layer in range(layers):
        g = torch.Generator(device="cuda").manual_seed(layer)
        if layout == "rows":
            k, v = (torch.randn(pages, size, heads, head_dim, generator=g, device="cuda").to(dtype) for _ in range(2))
        elif layout == "heads":
            k, v = (torch.randn(pages, heads, size, head_dim, generator=g, device="cuda").to(dtype).transpose(1, 2) for _ in range(2))
        elif layout == "pairs":
            both = torch.randn(pages, 2, size, heads, head_dim, generator=g, device="cuda").to(dtype)
            k, v = both[:, 0], both[:, 1]
        else:
            k, v = (torch.randn(pages, size, heads, head_dim + 4, generator=g, device="cuda").to(dtype)[..., :head_dim] for _ in range(2))
        caches.append(PagedCache(k, v))
    want = [(c.k.clone(), c.v.clone()) for c in caches]
    sources, destinations = [3, -1, 0, 22, 5, 7], [4, 6, 1, 21, -1, 7]
    for k, v in want:
        for a, b in zip(sources, destinations):
            if a >= 0 and b >= 0:
                k[b], v[b] = k[a].clone(), v[a].clone()
    backend.pages_copy(caches, torch.tensor(sources, dtype=torch.int32).cuda(), torch.tensor(destinations, dtype=torch.int32).cuda())
    backend.poll()
    for c, (k, v) in zip(caches, want):
        assert torch.equal(c.k, k) and torch.equal(c.v, v)
    backend.pages_copy(caches[0], torch.tensor([1, 2], dtype=torch.int32).cuda(), torch.tensor([23, 3], dtype=torch.int32).cuda())
    with pytest.raises(WB200Error):
        backend.poll()
    assert torch.equal(caches[0].k[3], want[0][0][2])


def test_copy_serves_more_caches_than_one_launch_holds(backend):
    caches = [PagedCache(*(torch.full((3, 2, 1, 8), float(i), device="cuda").bfloat16() for _ in range(2))) for i in range(70)]
    for i, c in enumerate(caches):
        c.k[0] = i + 0.5
    backend.pages_copy(caches, torch.tensor([0], dtype=torch.int32).cuda(), torch.tensor([2], dtype=torch.int32).cuda())
    assert all(torch.equal(c.k[2], c.k[0]) and torch.equal(c.k[1], torch.full_like(c.k[1], float(i))) for i, c in enumerate(caches))


def test_long_lists_of_pages_to_pass_over(backend):
    cache = PagedCache(*(torch.randn(9000, 1, 1, 64, device="cuda").bfloat16() for _ in range(2)))
    sources, destinations = torch.full((30000,), -1, dtype=torch.int32), torch.full((30000,), -1, dtype=torch.int32)
    at = torch.arange(0, 30000, 7)[:4000]
    order = torch.randperm(9000, generator=torch.Generator().manual_seed(1))
    sources[at], destinations[at] = order[:4000].int(), order[4000:8000].int()
    want = cache.k.clone()
    want[order[4000:8000]] = want[order[:4000]]
    backend.pages_copy(cache, sources.cuda(), destinations.cuda())
    assert torch.equal(cache.k, want)


def test_page_tables_in_place(backend):
    tables = PageTables(backend, 4, 8, 12, 4)
    cache = PagedCache.zeros(12, 4, 1, 8)
    assert int(tables.reserve(torch.tensor([5, 0, 9, 0], dtype=torch.int32).cuda())) == 0
    assert tables.table[0, :3].tolist() == [0, 1, -1] and tables.table[2, :4].tolist() == [2, 3, 4, -1] and tables.lengths.tolist() == [5, 0, 9, 0]
    cache.k[4] = 3.0
    assert int(tables.fork(torch.tensor([2], dtype=torch.int32).cuda(), torch.tensor([1], dtype=torch.int32).cuda(), [cache])) == 0
    assert tables.table[1, :4].tolist() == [2, 3, 5, -1] and tables.refs[:6].tolist() == [1, 1, 2, 2, 1, 1] and bool((cache.k[5] == 3.0).all())
    tables.free(torch.tensor([0, 2], dtype=torch.int32).cuda())
    assert tables.refs[:6].tolist() == [0, 0, 1, 1, 0, 1] and tables.lengths.tolist() == [0, 9, 0, 0]
    tables.compact([cache])
    assert tables.table[1, :3].tolist() == [2, 0, 1] and tables.refs[:6].tolist() == [1, 1, 1, 0, 0, 0] and bool((cache.k[1] == 3.0).all())
    backend.poll()


def test_poll_reports_one_thing_after_the_other(backend):
    """A wait that gave up and refused data, both pending: neither report is lost."""
    table, lengths, refs = state(12, 6, 100, 8, 3, fill=0.5)
    backend.pages_free(table, lengths, refs, torch.tensor([12], dtype=torch.int32).cuda(), 8)
    backend.selftest_bounded_wait(100_000)
    with pytest.raises(WB200Error, match="wait"):
        backend.poll()
    with pytest.raises(WB200Error, match="left out"):
        backend.poll()
    backend.poll()


@pytest.mark.parametrize("page", [-1, 100])
def test_fork_reports_a_last_page_outside_the_cache(backend, page):
    # the page that a child's own last page is to be copied from: without a report the child's rows would be whatever lies there
    table, lengths, refs = state(12, 6, 100, 8, 3, fill=0.5)
    lengths[0] = 0
    parent = max(range(1, 12), key=lambda s: int(lengths[s]))
    lengths[parent] = lengths[parent] // 8 * 8 - 3    # its last page holds five tokens
    table[parent, int(lengths[parent]) // 8] = page
    p, c = torch.tensor([parent], dtype=torch.int32).cuda(), torch.tensor([0], dtype=torch.int32).cuda()
    got = backend.pages_fork(table, lengths, refs, p, c, 8)
    assert int(got[5]) == 0 and got[3].tolist() == [-1]
    with pytest.raises(WB200Error, match="page number"):
        backend.poll()
    backend.poll()


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("pages,size", [(60, 8), (5000, 16), (70001, 4)])
def test_reserve_with_exactly_enough_and_too_few_pages(backend, pages, size, in_place):
    """Wants of all free pages and of three more, in pools of one and of many parts of the scan, spread over many sequences."""
    sequences, width = 40, pages // 16
    table, lengths, refs = state(sequences, width, pages, size, 5, fill=0.6)
    free = int((refs == 0).sum())
    for wanted_pages, outcome in ((free, 0), (free + 3, 3)):
        plain = ref.Pages(table, lengths, refs, size)
        have = [plain.count(s) for s in range(sequences)]
        wanted, spread = lengths.tolist(), wanted_pages
        for s in range(sequences):
            more = min(spread, width - have[s])
            if more:
                wanted[s] = (have[s] + more) * size - (s % size)
                spread -= more
        assert spread == 0
        wanted = torch.tensor(wanted, dtype=torch.int32).cuda()
        before = table.clone(), lengths.clone(), refs.clone()
        arrays = (table.clone(), lengths.clone(), refs.clone())
        got = backend.pages_reserve(*arrays, wanted, size, out=arrays if in_place else None)
        assert int(got[3]) == outcome
        if outcome:
            assert all(torch.equal(a, b) for a, b in zip(got[:3], before)) and all(torch.equal(a, b) for a, b in zip(arrays, before))
        else:
            assert plain.reserve(wanted) == 0 and int((got[2] == 0).sum()) == 0
            agree(plain, *got[:3])
    backend.poll()
