"""Attention over a paged KV cache against float64 (bounds: tests/paged_reference.attention)."""
import copy

import pytest
import torch

from tests import paged_reference as ref
from tests.test_gpu_rope import make_batch, make_cache
from vibe_compiler_b200.backend import WB200Error
from vibe_compiler_b200.paged_cache import PagedBatch, PagedCache, PageTables

pytestmark = pytest.mark.gpu


def spoil_unused(cache, batch, size):
    """NaN and infinities wherever no sequence has a key: behind the lengths and in pages nobody holds."""
    used = torch.zeros(cache.k.shape[:2], dtype=torch.bool)
    for row, n in zip(batch.page_table.cpu().tolist(), batch.key_lengths.tolist()):
        for j in range(n):
            used[row[j // size], j % size] = True
    used = used.cuda()
    cache.k[~used] = float("nan")
    cache.v[~used] = float("inf")


def agree(backend, q, cache, batch, scale, **options):
    lse = torch.full(q.shape[:2], 5.0, device="cuda")
    out = torch.full_like(q, 3.0)
    backend.attention_paged(q, cache, batch, scale, lse=lse, out=out, **options)
    backend.poll()
    want, want_lse, bound, bound_lse = ref.attention(q, cache.k, cache.v, batch.page_table, batch.key_lengths, batch.query_starts, scale, **options)
    tokens = int(batch.query_starts[-1])
    assert bool((out[tokens:] == 3.0).all()) and bool((lse[tokens:] == 5.0).all())
    got, want, bound = out[:tokens].double(), want[:tokens], bound[:tokens]
    assert torch.equal(got.isnan(), want.isnan())
    excess = ((got - want).abs() - bound).nan_to_num(nan=-1.0)
    assert excess.max().item() <= 0, excess.max().item()
    got, want, bound = lse[:tokens].double(), want_lse[:tokens], bound_lse[:tokens]
    assert torch.equal(got.isinf(), want.isinf())
    excess = ((got - want).abs() - bound)[~want.isinf()]
    assert excess.numel() == 0 or excess.max().item() <= 0, excess.max().item()
    return out


# (keys with the new tokens, new tokens, page size, query heads, KV heads, head_dim)
CASES = [
    ([1], [1], 16, 1, 1, 128), ([17], [1], 16, 4, 4, 64), ([700, 64, 65, 2000, 0, 1], [1] * 6, 16, 28, 4, 128),
    ([129, 5, 300, 0], [1, 0, 1, 0], 32, 32, 8, 128), ([4097, 33], [1, 1], 128, 8, 8, 64), ([513, 900], [1, 1], 48, 16, 1, 128),
    ([40, 300], [8, 3], 16, 16, 4, 64), ([257, 128], [5, 9], 64, 28, 4, 128),                     # a few tokens each
    ([128], [128], 16, 4, 1, 128), ([129], [129], 32, 2, 2, 128), ([300, 77], [300, 41], 16, 32, 8, 128),   # prompts
    ([1000, 640, 2, 333], [250, 1, 2, 333], 128, 8, 2, 128), ([700, 1500], [260, 90], 64, 6, 2, 64), ([513], [200], 24, 5, 1, 128),
    ([2500, 90, 1200], [64, 1, 1], 32, 28, 4, 128), ([600, 600], [33, 65], 100, 7, 7, 128), ([350], [150], 3, 4, 2, 128),
    ([77, 300], [77, 20], 16, 4, 2, 80), ([50], [3], 7, 3, 1, 256), ([90], [90], 16, 2, 2, 8), ([60], [60], 16, 40, 1, 64),
    ([200, 150], [30, 150], 256, 64, 1, 128), ([300], [5], 16, 160, 1, 128), ([400], [130], 8, 12, 2, 64)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lengths,news,size,hq,hk,head_dim", CASES)
def test_attention_matches_float64(backend, dtype, causal, lengths, news, size, hq, hk, head_dim):
    pages = sum(-(-n // size) for n in lengths) + 3
    cache = make_cache(pages, size, hk, head_dim, dtype, "rows", 1)
    batch, tokens = make_batch(lengths, news, size, pages, 2, spare_rows=3)
    spoil_unused(cache, batch, size)
    q = torch.randn(tokens, hq, head_dim, generator=torch.Generator().manual_seed(3)).to(dtype).cuda()
    wide, _ = make_batch(lengths, news, size, pages, 2, width=65536 // size + 2)     # room for longer sequences
    for max_query, table in ((0, batch.page_table), (1, batch.page_table), (max(news), batch.page_table), (1, wide.page_table), (0, wide.page_table)):
        hinted = PagedBatch(table, batch.key_lengths, batch.query_starts, max_query=max_query)      # a hint: right, wrong or missing
        agree(backend, q, cache, hinted, head_dim ** -0.5, causal=causal, zero_fully_masked=max_query == 1)


@pytest.mark.parametrize("layout", ["heads", "pairs"])
@pytest.mark.parametrize("lengths,news", [([300, 1000], [1, 1]), ([300, 1000], [200, 150])])
def test_layouts_and_strides(backend, layout, lengths, news):
    size, hq, hk, d = 32, 8, 2, 128
    cache = make_cache(50, size, hk, d, torch.bfloat16, layout, 1)
    batch, tokens = make_batch(lengths, news, size, 50, 2)
    fused = torch.randn(tokens, hq + 2 * hk, d, generator=torch.Generator().manual_seed(5)).bfloat16().cuda()
    want = backend.attention_paged(fused[:, :hq].contiguous(), cache, batch, 0.1)
    agree(backend, fused[:, :hq], cache, batch, 0.1)
    out = torch.empty(hq, tokens, d, dtype=torch.bfloat16, device="cuda").transpose(0, 1)
    backend.attention_paged(fused[:, :hq], cache, batch, 0.1, out=out)
    assert torch.equal(out, want)
    wide = torch.full((2, batch.page_table.shape[1] + 5), 10 ** 6, dtype=torch.int32, device="cuda")
    wide[:, :batch.page_table.shape[1]] = batch.page_table
    view = PagedBatch(wide[:, :batch.page_table.shape[1]], batch.key_lengths, batch.query_starts)
    assert torch.equal(backend.attention_paged(fused[:, :hq], cache, view, 0.1), want)
    backend.poll()


@pytest.mark.parametrize("lengths,news", [([300, 1000], [1, 1]), ([300, 1000], [200, 150])])
@pytest.mark.parametrize("order", ["queries off 16 bytes", "output off 16 bytes", "heads outside tokens", "V in another order than K",
                                   "pages inside rows", "cache off 16 bytes"])
def test_orders_that_need_another_kernel(backend, lengths, news, order):
    size, hq, hk, d = 32, 8, 2, 128
    cache = make_cache(50, size, hk, d, torch.float16, "rows", 1)
    batch, tokens = make_batch(lengths, news, size, 50, 2)
    q = torch.randn(tokens, hq, d, generator=torch.Generator().manual_seed(5)).half().cuda()

    def apart(t, shift):                              # the same values, `shift` elements into a buffer
        buffer = torch.zeros(t.numel() + shift, dtype=t.dtype, device="cuda")
        view = buffer[shift:].view(t.shape)
        view.copy_(t)
        return view
    out = None
    if order == "queries off 16 bytes":
        q = apart(q, 3)
    elif order == "output off 16 bytes":
        out = apart(torch.zeros_like(q), 1)
    elif order == "heads outside tokens":
        q = q.transpose(0, 1).contiguous().transpose(0, 1)
    elif order == "V in another order than K":
        cache = PagedCache(cache.k, cache.v.transpose(1, 2).contiguous().transpose(1, 2))
    elif order == "pages inside rows":
        cache = PagedCache(*(t.transpose(0, 1).contiguous().transpose(0, 1) for t in (cache.k, cache.v)))
    else:
        cache = PagedCache(apart(cache.k, 4), apart(cache.v, 4))
    want, _, bound, _ = ref.attention(q, cache.k, cache.v, batch.page_table, batch.key_lengths, batch.query_starts, 0.1)
    got = backend.attention_paged(q, cache, batch, 0.1, out=out)
    backend.poll()
    assert bool(((got.double() - want).abs() <= bound).all())


def test_more_sequences_than_a_block_stages(backend):
    count = 5000
    news = [0] * count
    news[17], news[4999], news[3000] = 40, 1, 9
    lengths = [0] * count
    lengths[17], lengths[4999], lengths[3000], lengths[4] = 70, 33, 9, 16
    cache = make_cache(20, 16, 2, 128, torch.bfloat16, "rows", 1)
    batch, tokens = make_batch(lengths, news, 16, 20, 2)
    agree(backend, torch.randn(tokens, 8, 128, device="cuda").bfloat16(), cache, batch, 0.1)
    few = PagedBatch(batch.page_table[:4000], batch.key_lengths[:4000].contiguous(), batch.query_starts[:4001].contiguous())
    agree(backend, torch.randn(tokens, 8, 128, device="cuda").bfloat16(), cache, few, 0.1)


def test_one_page_in_many_places(backend):
    # a sequence may list a page more than once: 40 thousand keys over three pages
    cache = make_cache(3, 128, 2, 128, torch.bfloat16, "rows", 1)
    table = torch.arange(320, dtype=torch.int32, device="cuda")[None, :] % 3
    for n in (1, 70):
        batch = PagedBatch(table, torch.tensor([40900], dtype=torch.int32, device="cuda"), torch.tensor([0, n], dtype=torch.int32, device="cuda"))
        agree(backend, torch.randn(n, 8, 128, device="cuda").bfloat16(), cache, batch, 0.1)


def test_empty_calls(backend):
    cache = make_cache(4, 16, 2, 128, torch.bfloat16, "rows", 1)
    batch, _ = make_batch([20, 0], [0, 0], 16, 4, 2)
    assert backend.attention_paged(torch.empty(0, 8, 128, dtype=torch.bfloat16, device="cuda"), cache, batch, 0.1).shape == (0, 8, 128)
    untouched = torch.full((3, 8, 128), 2.0, dtype=torch.bfloat16, device="cuda")
    backend.attention_paged(torch.zeros_like(untouched), cache, batch, 0.1, out=untouched)
    backend.poll()
    assert bool((untouched == 2.0).all())


@pytest.mark.parametrize("lengths,news", [([90, 40], [1, 1]), ([90, 40, 10], [60, 50, 30])])
def test_rows_without_keys(backend, lengths, news):
    # more new tokens than keys: the first ones stand in front of key 0
    lengths = [n // 2 for n in lengths]
    cache = make_cache(20, 16, 2, 128, torch.float16, "rows", 1)
    batch, tokens = make_batch(lengths, news, 16, 20, 2)
    spoil_unused(cache, batch, 16)
    q = torch.randn(tokens, 8, 128, device="cuda").half()
    for zero in (False, True):
        agree(backend, q, cache, batch, 0.1, zero_fully_masked=zero)


@pytest.mark.parametrize("magnitude", [30.0, 3e3])
def test_large_scores(backend, magnitude):
    cache = make_cache(50, 16, 2, 128, torch.bfloat16, "rows", 1)
    cache.k.mul_(magnitude)
    batch, tokens = make_batch([500, 130], [40, 1], 16, 50, 2)
    q = torch.randn(tokens, 8, 128, generator=torch.Generator().manual_seed(5)).bfloat16().cuda()
    agree(backend, q, cache, batch, 128 ** -0.5)


def test_results_do_not_depend_on_where_the_pages_lie_or_on_the_run(backend):
    size, lengths, news = 16, [900, 5000, 33, 260], [1, 1, 1, 1]
    cache = make_cache(420, size, 4, 128, torch.bfloat16, "rows", 1)
    batch, tokens = make_batch(lengths, news, size, 420, 2)
    q = torch.randn(tokens, 28, 128, device="cuda").bfloat16()
    want = backend.attention_paged(q, cache, batch, 0.09)
    for _ in range(5):
        assert torch.equal(backend.attention_paged(q, cache, batch, 0.09), want)
    order = torch.randperm(420, device="cuda")
    moved = PagedCache(torch.empty_like(cache.k), torch.empty_like(cache.v))
    moved.k[order], moved.v[order] = cache.k, cache.v
    table = torch.where(batch.page_table >= 0, order[batch.page_table.clamp(min=0).long()].int(), batch.page_table)
    assert torch.equal(backend.attention_paged(q, moved, PagedBatch(table, batch.key_lengths, batch.query_starts), 0.09), want)


@pytest.mark.parametrize("news", [[1, 1], [80, 70]])
@pytest.mark.parametrize("fault", ["page too large", "page negative", "length beyond the table", "tokens beyond the rows"])
def test_bad_device_data_is_left_out_and_reported(backend, news, fault):
    cache = make_cache(30, 16, 2, 128, torch.bfloat16, "rows", 1)
    batch, tokens = make_batch([200, 150], news, 16, 30, 2)
    q = torch.randn(tokens, 8, 128, device="cuda").bfloat16()
    # The other sequence's rows are right; where its keys are cut, and so the order of its sums, follows what is left of the batch.
    want, _, bound, _ = ref.attention(q, cache.k, cache.v, batch.page_table, batch.key_lengths, batch.query_starts, 0.1)
    if fault.startswith("page"):
        batch.page_table[1, 3] = 30 if fault == "page too large" else -7
    elif fault.startswith("length"):
        batch.key_lengths[1] = 5000
    else:
        batch.query_starts[2] = tokens + 40
    got = backend.attention_paged(q, cache, batch, 0.1)
    with pytest.raises(WB200Error):
        backend.poll()
    assert bool(((got.double() - want).abs() <= bound)[:news[0]].all())
    backend.poll()


def test_a_captured_call_follows_the_lengths_on_the_device(backend):
    size = 16
    cache = make_cache(600, size, 4, 128, torch.bfloat16, "rows", 1)
    long, tokens = make_batch([4000, 900, 2000], [1, 1, 1], size, 600, 2)
    q = torch.randn(tokens, 28, 128, device="cuda").bfloat16()
    batch = PagedBatch(long.page_table.clone(), long.key_lengths.clone(), long.query_starts.clone(), max_query=1)
    backend.attention_paged(q, cache, batch, 0.1)
    graphs, outs = [], []
    for _ in range(2):                               # two graphs of the same call, replayed at the same time
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(backend.attention_paged(q, cache, batch, 0.1))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for lengths in ([4000, 900, 2000], [17, 4000, 1], [3, 5, 3999]):
        batch.key_lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
        wide, _ = make_batch(lengths, [1, 1, 1], size, 600, 9, width=batch.page_table.shape[1])
        batch.page_table.copy_(wide.page_table)
        torch.cuda.synchronize()
        for _ in range(3):
            for graph, stream in zip(graphs, streams):
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        want = backend.attention_paged(q, cache, batch, 0.1)
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want)
    backend.poll()


@pytest.mark.parametrize("news", [[1, 1, 1], [200, 1, 64]])
def test_calls_on_two_streams_at_once(backend, news):
    cache = make_cache(600, 16, 4, 128, torch.float16, "rows", 1)
    batch, tokens = make_batch([4000, 900, 2000], news, 16, 600, 2)
    qs = [torch.randn(tokens, 28, 128, device="cuda").half() for _ in range(2)]
    wants = [backend.attention_paged(q, cache, batch, 0.1) for q in qs]
    streams = [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    results = [[], []]
    for _ in range(10):
        for i, stream in enumerate(streams):
            results[i].append(backend.attention_paged(qs[i], cache, batch, 0.1, stream=stream.cuda_stream))
    torch.cuda.synchronize()
    for want, got in zip(wants, results):
        assert all(torch.equal(want, g) for g in got)


def test_a_cache_beyond_32_bit_offsets(backend):
    pages, size, hk, d = 20000, 128, 8, 128          # 2.6e9 elements each of K and V
    k, v = (torch.zeros(pages, size, hk, d, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    cache = PagedCache(k, v)
    picked = torch.tensor([[19999, 3, 17000], [18888, 16500, 1]], dtype=torch.int32, device="cuda")
    for page in picked.flatten().tolist():
        k[page], v[page] = torch.randn(size, hk, d, device="cuda").bfloat16(), torch.randn(size, hk, d, device="cuda").bfloat16()
    for news in ([1, 1], [100, 70]):
        batch = PagedBatch(picked, torch.tensor([300, 384], dtype=torch.int32, device="cuda"),
                           torch.tensor([0, news[0], sum(news)], dtype=torch.int32, device="cuda"))
        agree(backend, torch.randn(sum(news), 32, d, device="cuda").bfloat16(), cache, batch, 0.1)
        qkv = torch.randn(sum(news), (32 + 2 * hk) * d, device="cuda").bfloat16()
        backend.rope_append(qkv, cache, batch, None, q_heads=32)
        assert torch.equal(ref.gathered(v, picked[0], 300, size)[300 - news[0]:], qkv.view(-1, 48, d)[:news[0], 40:])
    tables = torch.tensor([19999, 17000], dtype=torch.int32, device="cuda"), torch.tensor([5, 19998], dtype=torch.int32, device="cuda")
    backend.pages_copy(cache, *tables)
    assert torch.equal(k[5], k[19999]) and torch.equal(v[19998], v[17000])
    backend.poll()


def test_a_serving_run(backend):
    """Prompts in pieces, decoding, a fork, a freed sequence and moved pages, against the decoder layer over whole sequences."""
    from vibe_compiler_b200.decoder_layer import LayerConfig, ShardedDecoderLayer, random_weights
    cfg = LayerConfig(d_model=512, q_heads=8, kv_heads=2, head_dim=128, ffn=768)
    layer = ShardedDecoderLayer(backend, cfg, random_weights(cfg))
    size, sequences = 16, 5
    tables, cache = PageTables(backend, sequences, 24, 60, size), PagedCache.zeros(60, size, 2, 128)
    g = torch.Generator().manual_seed(11)
    texts = {s: torch.randn(n, 512, generator=g).bfloat16().cuda() for s, n in ((0, 150), (1, 37), (3, 200))}
    done, outputs = {s: 0 for s in texts}, {s: [] for s in texts}

    def step(counts):
        lengths = [done.get(s, 0) + counts.get(s, 0) for s in range(sequences)]
        assert int(tables.reserve(torch.tensor(lengths, dtype=torch.int32).cuda())) == 0
        starts = [0]
        for s in range(sequences):
            starts.append(starts[-1] + counts.get(s, 0))
        x = torch.cat([texts[s][done[s]:done[s] + counts[s]] for s in range(sequences) if counts.get(s)])
        batch = PagedBatch(tables.table, tables.lengths, torch.tensor(starts, dtype=torch.int32).cuda(), max_query=max(counts.values()))
        y = layer.forward_paged(x, cache, batch)
        for s, n in counts.items():
            outputs[s].append(y[starts[s]:starts[s] + n])
            done[s] += n

    step({0: 70, 1: 20, 3: 130})
    step({0: 1, 1: 1, 3: 33})                        # decoding next to a piece of a prompt
    texts[4], done[4] = torch.cat([texts[3][:done[3]], torch.randn(30, 512, generator=g).bfloat16().cuda()]), done[3]
    outputs[4] = list(outputs[3])
    assert int(tables.fork(torch.tensor([3], dtype=torch.int32).cuda(), torch.tensor([4], dtype=torch.int32).cuda(), [cache])) == 0
    for _ in range(5):
        step({0: 1, 1: 1, 3: 1, 4: 1})
    tables.free(torch.tensor([1], dtype=torch.int32).cuda())
    done[1] = 0
    finished = outputs.pop(1)
    tables.compact([cache])
    for _ in range(3):
        step({0: 2, 3: 1, 4: 3})
    backend.poll()
    outputs[1] = finished
    for s, parts in outputs.items():
        got = torch.cat(parts)
        text = torch.nn.functional.pad(texts[s][:len(got)], (0, 0, 0, -len(got) % 8))       # the layer takes rows by eights
        whole = layer.forward(text[None])[0, :len(got)]
        # both round every stage to bf16 on the way; the suite's bound for the layer
        assert (got.double() - whole.double()).abs().max().item() <= 1e-2 * whole.double().abs().max().item()


@pytest.mark.parametrize("sequences", [3, 40])
def test_a_captured_serving_step(backend, sequences):
    """One decoding step - room, cache writes, attention, the layer around them - captured once and replayed: each replay takes
    the next token of every sequence, as the lengths, tables and page counts on the device go on."""
    from vibe_compiler_b200.decoder_layer import LayerConfig, ShardedDecoderLayer, random_weights
    cfg = LayerConfig(d_model=512, q_heads=8, kv_heads=2, head_dim=128, ffn=768)
    layer = ShardedDecoderLayer(backend, cfg, random_weights(cfg))
    size, steps, pages = 16, 20, 8 * sequences
    g = torch.Generator().manual_seed(3)
    prompts = [int(n) for n in torch.randint(1, 90, (sequences,), generator=g)]
    texts = [torch.randn(n + steps, 512, generator=g).bfloat16().cuda() for n in prompts]

    def begin():
        tables, cache = PageTables(backend, sequences, 40, pages, size), PagedCache.zeros(pages, size, 2, 128)
        assert int(tables.reserve(torch.tensor(prompts, dtype=torch.int32).cuda())) == 0
        starts = torch.tensor([0] + prompts, dtype=torch.int32).cumsum(0).int().cuda()
        layer.forward_paged(torch.cat([t[:n] for t, n in zip(texts, prompts)]), cache, PagedBatch(tables.table, tables.lengths, starts, max_query=max(prompts)))
        return tables, cache

    one_each = torch.arange(sequences + 1, dtype=torch.int32, device="cuda")

    def step(tables, cache, x):
        result = tables.reserve(tables.lengths + 1)
        return layer.forward_paged(x, cache, PagedBatch(tables.table, tables.lengths, one_each, max_query=1)), result
    tokens = [torch.stack([t[n + i] for t, n in zip(texts, prompts)]) for i in range(steps)]
    state = begin()
    want = [step(*state, x)[0].clone() for x in tokens]
    warm = begin()
    step(*warm, tokens[0])
    state, x = begin(), tokens[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, result = step(*state, x)
    for i in range(steps):
        x.copy_(tokens[i])
        graph.replay()
        assert int(result) == 0 and torch.equal(y, want[i])
    backend.poll()
    assert state[0].lengths.tolist() == [n + steps for n in prompts]


# (sequences, most new tokens, most keys in front, KV heads, group, head_dim): more heads than a warp's lanes, more sequences than a
# look at every 32nd finds in one go, no work in front of and between the sequences, fewer shares than SMs, one item for all SMs.
@pytest.mark.parametrize("sequences,news,front,hk,group,head_dim", [
    (5, 30, 200, 33, 1, 64), (3, 20, 90, 70, 1, 64), (1500, 9, 20, 2, 4, 64), (1100, 3, 40, 1, 8, 128), (2, 9, 30, 1, 4, 64),
    (1, 40, 12000, 1, 8, 128), (1, 2, 20000, 1, 2, 64), (40, 70, 600, 3, 5, 128)])
def test_work_is_shared_out_whole(backend, sequences, news, front, hk, group, head_dim):
    rng = torch.Generator().manual_seed(sequences)
    new = torch.randint(0, news + 1, (sequences,), generator=rng).tolist()
    new[0], new[-1] = (0 if sequences > 2 else news), news
    lengths = [n + int(torch.randint(0, front + 1, (1,), generator=rng)) if n else 0 for n in new]
    lengths[-1] = front + news
    size = 16
    pages = sum(-(-n // size) for n in lengths) + 3
    cache = make_cache(pages, size, hk, head_dim, torch.bfloat16, "rows", 1)
    batch, tokens = make_batch(lengths, new, size, pages, 2, spare_rows=3)
    q = torch.randn(tokens, hk * group, head_dim, generator=rng).bfloat16().cuda()
    for max_query in (0, 1, news):
        agree(backend, q, cache, PagedBatch(batch.page_table, batch.key_lengths, batch.query_starts, max_query=max_query), head_dim ** -0.5)


@pytest.mark.parametrize("stride", [0, 64, 128])
@pytest.mark.parametrize("news", [[9, 3], [200, 70]])
def test_one_query_head_of_any_token_stride(backend, news, stride):
    # queries that share memory, all of one row or half of the one before, are read like any others
    cache = make_cache(50, 32, 1, 128, torch.bfloat16, "rows", 1)
    batch, tokens = make_batch([300, 500], news, 32, 50, 2)
    buffer = torch.randn(tokens * 128, generator=torch.Generator().manual_seed(5)).bfloat16().cuda()
    agree(backend, buffer.as_strided((tokens, 1, 128), (stride, 128, 1)), cache, batch, 0.1)


def test_a_decoding_step_of_the_layer_takes_the_decoding_kernel(backend):
    """Without the caller's word on the longest chunk, 3 tokens of 3 sequences are one each; a range that ends behind them is reported."""
    from vibe_compiler_b200.decoder_layer import LayerConfig, ShardedDecoderLayer, random_weights
    cfg = LayerConfig(d_model=512, q_heads=8, kv_heads=2, head_dim=128, ffn=768)
    layer = ShardedDecoderLayer(backend, cfg, random_weights(cfg))
    cache = make_cache(30, 16, 2, 128, torch.bfloat16, "rows", 1)
    batch, tokens = make_batch([90, 40, 200], [1, 1, 1], 16, 30, 2)
    x = torch.randn(tokens, 512, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    launches, results = [], []
    for max_query in (1, 0):
        before = backend.launch_count
        hinted = PagedBatch(batch.page_table, batch.key_lengths, batch.query_starts, max_query=max_query)
        results.append(layer.forward_paged(x, cache, hinted))
        launches.append(backend.launch_count - before)
    assert launches[0] == launches[1] and torch.equal(*results)
    backend.poll()
    batch.query_starts[3] += 2
    layer.forward_paged(x, cache, batch)
    with pytest.raises(WB200Error):
        backend.poll()
    backend.poll()


# (keys, new tokens, query heads): units and items whole, halved, cut over CTAs, and taken by clusters; the last by the general kernel
@pytest.mark.parametrize("lengths,news,hq,hk,head_dim", [
    ([700, 90], [1, 1], 8, 2, 128), ([9000] * 12, [1] * 12, 8, 8, 64), ([300, 260], [200, 250], 4, 2, 128), ([500, 300], [40, 9], 4, 2, 64),
    ([20000], [60], 4, 2, 128), ([9000], [500], 4, 1, 64), ([150, 90], [70, 1], 2, 1, 72)])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_scores_that_are_no_numbers(backend, lengths, news, hq, hk, head_dim, value):
    """A NaN or infinite score among the keys that a row sees makes what the definition makes of it: NaN, or for -inf a key without
    weight. Rows that do not see it, of the same tile or of another sequence, keep their values."""
    size = 16
    cache = make_cache(sum(-(-n // size) for n in lengths) + 3, size, hk, head_dim, torch.bfloat16, "rows", 1)
    batch, tokens = make_batch(lengths, news, size, cache.k.shape[0], 2)
    q = torch.randn(tokens, hq, head_dim, generator=torch.Generator().manual_seed(3)).bfloat16().cuda()
    q[..., 0] = q[..., 0].abs() + 0.5                 # what meets the infinity is positive

    def of(key):
        return batch.page_table[0].long()[key // size], key % size
    bad = lengths[0] - news[0] // 2 - 1               # half of the first sequence's tokens see this key
    cache.k[(*of(torch.tensor(bad, device="cuda")), slice(None), 0)] = value
    sees = torch.zeros(tokens, dtype=torch.bool, device="cuda")
    sees[bad - (lengths[0] - news[0]):news[0]] = True
    expected = ref.attention(q, cache.k, cache.v, batch.page_table, batch.key_lengths, batch.query_starts, 0.1)
    if value == -float("inf"):
        # for the rows that see it: the same without the key, those behind it one place further in front
        k, v, fewer = cache.k.clone(), cache.v.clone(), batch.key_lengths.clone()
        behind = torch.arange(bad + 1, lengths[0], device="cuda")
        k[of(behind - 1)], v[of(behind - 1)] = cache.k[of(behind)], cache.v[of(behind)]
        fewer[0] -= 1
        for whole, seen in zip(expected, ref.attention(q, k, v, batch.page_table, fewer, batch.query_starts, 0.1)):
            whole[sees] = seen[sees]
    want, want_lse, bound, bound_lse = expected
    for max_query in (0, 1, max(news)):
        out, lse = torch.full_like(q, 3.0), torch.full(q.shape[:2], 5.0, device="cuda")
        hinted = PagedBatch(batch.page_table, batch.key_lengths, batch.query_starts, max_query=max_query)
        backend.attention_paged(q, cache, hinted, 0.1, out=out, lse=lse)
        backend.poll()
        rows = torch.ones_like(sees) if value == -float("inf") else ~sees
        assert bool(((out.double() - want).abs() <= bound)[rows].all()) and bool(((lse.double() - want_lse).abs() <= bound_lse)[rows].all())
        assert bool(out[~rows].isnan().all()) and not bool(lse[~rows].isfinite().any())


def test_copied_handles_describe_the_tensors_they_hold(backend):
    """A copy, or an object sent to another process, has tensors of its own: the addresses that a call passes on have to be theirs."""
    cache = make_cache(20, 16, 2, 128, torch.bfloat16, "rows", 1)
    batch, _ = make_batch([90, 40], [1, 1], 16, 20, 2)
    batch = PagedBatch(batch.page_table, batch.key_lengths, batch.query_starts, max_query=7)
    for again in (copy.copy, copy.deepcopy):
        other, d = again(batch), again(batch)._desc(2)
        for name in ("page_table", "key_lengths", "query_starts"):
            assert torch.equal(getattr(other, name), getattr(batch, name)) and getattr(other._desc(2), name) == getattr(other, name).data_ptr()
        assert (d.sequences, d.max_query, other.max_query) == (2, 7, 7)
        other = again(cache)
        assert (other._desc.k, other._desc.v) == (other.k.data_ptr(), other.v.data_ptr()) and torch.equal(other.k, cache.k)
    for name in ("page_table", "key_lengths", "query_starts"):      # a tensor put in another's place is the one that is read
        setattr(batch, name, getattr(batch, name).clone())
        assert getattr(batch._desc(2), name) == getattr(batch, name).data_ptr()
        with pytest.raises(ValueError):
            setattr(batch, name, getattr(batch, name).long())
    cache.k, cache.v, batch.max_query = cache.k.clone(), cache.v.clone(), 9
    assert (cache._desc.k, cache._desc.v, batch._desc(2).max_query) == (cache.k.data_ptr(), cache.v.data_ptr(), 9)
    before = batch.key_lengths.data_ptr()
    batch.key_lengths += 1
    assert batch.key_lengths.data_ptr() == before and batch.key_lengths.tolist() == [91, 41]
    with pytest.raises(ValueError):
        cache.k = cache.k[:10]


def test_rejected_drafts_are_written_over(backend):
    """Two of five drafted tokens stay: the next ones go over the others' rows, their room reserved all along."""
    size, hq, hk, d = 4, 4, 2, 64
    tables, cache = PageTables(backend, 1, 20, 30, size), PagedCache.zeros(30, size, hk, d)
    rows = torch.randn(60, (hq + 2 * hk) * d, generator=torch.Generator().manual_seed(2)).bfloat16().cuda()
    keys, kept = torch.zeros(1, dtype=torch.int32, device="cuda"), []      # the true number of keys; the rows behind them

    def step(new, stay):
        keys.fill_(len(kept) + len(new))
        assert int(tables.reserve(keys)) == 0
        batch = PagedBatch(tables.table, keys, torch.tensor([0, len(new)], dtype=torch.int32, device="cuda"))
        q = backend.rope_append(rows[new], cache, batch, None, q_heads=hq)
        out = backend.attention_paged(q, cache, batch, 0.125)
        seen = rows[kept + new].view(-1, hq + 2 * hk, d)
        plain = PagedCache(*(t.contiguous()[None] for t in (seen[:, hq:hq + hk], seen[:, hq + hk:])))
        one = PagedBatch(torch.zeros(1, 1, dtype=torch.int32, device="cuda"), keys, batch.query_starts)
        want, _, bound, _ = ref.attention(q, plain.k, plain.v, one.page_table, keys, batch.query_starts, 0.125)
        assert bool(((out.double() - want).abs() <= bound).all())
        kept.extend(new[:stay])

    step(list(range(9)), 9)
    step([10, 11, 12, 13, 14], 2)
    step([20, 21], 1)
    step([30, 31, 32, 33, 34, 35], 6)
    backend.poll()
    assert int(tables.refs.sum()) == -(-18 // size) and len(kept) == 18
