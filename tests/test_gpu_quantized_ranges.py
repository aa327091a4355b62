"""Attention over a cache in four bits at the ends of what its types hold: the few-rows kernel held to its own bound, that of scores
kept to f32 and of probabilities, weighed by the steps, in f16 (tests/quantized_reference.attention, "rows")."""
import pytest
import torch

from tests import quantized_reference as quant
from tests.test_gpu_quantized_cache import make_quantized, spoil_unused
from tests.test_gpu_rope import make_batch
from vibe_compiler_b200.paged_cache import PagedBatch, PagedCache, QuantizedCache

pytestmark = pytest.mark.gpu


def near(backend, q, cache, batch, scale, kernel="rows", vanishes=0.0, **options):
    """`kernel`: whose bound the rows have to keep, one for all or one for each token. `vanishes`: added to it, an element each."""
    lse = torch.full(q.shape[:2], 5.0, device="cuda")
    out = backend.attention_paged(q, cache, batch, scale, lse=lse, **options)
    backend.poll()
    of = {name: quant.attention(q, cache, batch, scale, kernel=name, **options) for name in ({kernel} if isinstance(kernel, str) else set(kernel))}
    for token in range(int(batch.query_starts[-1])):
        want, want_lse, bound, bound_lse = (t[token] for t in of[kernel if isinstance(kernel, str) else kernel[token]])
        got, got_lse = out[token].double(), lse[token].double()
        assert torch.equal(got.isnan(), want.isnan()) and bool(got[~want.isnan()].isfinite().all()), token
        excess = ((got - want).abs() - bound - vanishes).nan_to_num(nan=-1.0)
        assert excess.max().item() <= 0, (token, excess.max().item())
        assert torch.equal(got_lse.isinf(), want_lse.isinf()), token
        excess = ((got_lse - want_lse).abs() - bound_lse)[~want_lse.isinf()]
        assert excess.numel() == 0 or excess.max().item() <= 0, (token, excess.max().item())
    return out


def of_the_step(batch, news):
    return PagedBatch(batch.page_table, batch.key_lengths, batch.query_starts, max_query=max(news))


@pytest.mark.parametrize("hq,hk,head_dim,news", [(8, 2, 128, [1, 1]), (16, 2, 128, [1, 1]), (16, 2, 128, [2, 1]), (8, 2, 64, [2, 4])])
@pytest.mark.parametrize("signs", ["both", "one"])
@pytest.mark.parametrize("exponent,scale", [(118, 0.088), (121, 0.088), (124, 0.088), (100, 0.088), (-100, 0.088), (-120, 0.088), (6, 1e38)])
def test_queries_of_any_size_whose_scores_are_finite(backend, hq, hk, head_dim, news, signs, exponent, scale):
    """Queries near the type's largest numbers, whose sums would leave f32, on keys as small, and the other way around; one row of an
    ordinary size beside them."""
    cache = make_quantized(50, 16, hk, head_dim, torch.bfloat16)
    cache.k_steps.mul_(2.0 ** -exponent if scale < 1e38 else 2.0 ** -124)            # scores of about one
    batch, tokens = make_batch([500, 130], news, 16, 50, 2)
    q = torch.randn(tokens, hq, head_dim, generator=torch.Generator().manual_seed(5))
    q = (q.abs() if signs == "one" else q).bfloat16().cuda() * 2.0 ** exponent
    if scale == 1e38:
        q *= 2.0 ** -10                              # 2^-124 2^-4 1e38: about one
    q[0, 1] = 1.0
    batch = of_the_step(batch, news)
    near(backend, q, cache, batch, scale)


def vanishing(cache, q_heads, keys):
    """What the products of probability and step that f16 cannot hold are off by, an element of the result: 2^-25 each at most, in a unit
    that brings the group's largest step to 2^5 and more, for codes that are 8 away from the middle; a row's sum is 1 and more."""
    most = cache.v_steps[..., 0].double().amax((0, 1))                          # [kv_heads, groups]
    return (most * (keys * 2.0 ** -27)).repeat_interleave(64, -1).repeat_interleave(q_heads // cache.shape[2], 0)


ROWS = [(8, 2, [1, 1]), (16, 2, [1, 1]), (16, 2, [2, 1])]                       # four, eight and sixteen rows to a tile


@pytest.mark.parametrize("dtype,exponent", [(torch.bfloat16, 12), (torch.bfloat16, 20), (torch.bfloat16, 100), (torch.float16, 8)])
@pytest.mark.parametrize("first_is_small", [True, False])
@pytest.mark.parametrize("hq,hk,news", ROWS)
def test_groups_of_a_row_may_differ_in_size(backend, dtype, exponent, first_is_small, hq, hk, news):
    """The values of one group of 64 elements 2^(2 exponent) times the other's: each to its own bound."""
    cache = make_quantized(50, 16, hk, 128, dtype)
    sizes = (2.0 ** -exponent, 2.0 ** exponent) if first_is_small else (2.0 ** exponent, 2.0 ** -exponent)
    for group, size in enumerate(sizes):
        cache.v_steps[..., group, :] *= size
    batch, tokens = make_batch([500, 130], news, 16, 50, 2)
    q = torch.randn(tokens, hq, 128, generator=torch.Generator().manual_seed(5)).to(dtype).cuda()
    batch = of_the_step(batch, news)
    near(backend, q, cache, batch, 128 ** -0.5, vanishes=vanishing(cache, hq, 500))


@pytest.mark.parametrize("dtype,exponent", [(torch.bfloat16, 12), (torch.float16, 8)])
@pytest.mark.parametrize("hq,hk,news", ROWS)
def test_means_of_many_values_in_groups_of_different_sizes(backend, dtype, exponent, hq, hk, news):
    """As test_means_of_many_values_keep_their_digits, with its bound for each group."""
    cache = make_quantized(500, 64, hk, 128, dtype, seed=8)
    cache.v_steps[..., 0, :] *= 2.0 ** -exponent
    cache.v_steps[..., 1, :] *= 2.0 ** exponent
    batch, tokens = make_batch([30000, 1000], news, 64, 500, 2)
    q = torch.randn(tokens, hq, 128, generator=torch.Generator().manual_seed(3)).to(dtype).cuda()
    batch = of_the_step(batch, news)
    got = backend.attention_paged(q, cache, batch, 128 ** -0.5).double()
    backend.poll()
    want = quant.attention(q, cache, batch, 128 ** -0.5)[0]
    u = torch.finfo(dtype).eps / 2
    for group in (slice(0, 64), slice(64, 128)):
        for a, b in zip(got[..., group], want[..., group]):
            assert (a - b).norm() <= (2.0 ** -11 / 3 ** 0.5 + 1.6e-3 + u / 3 ** 0.5) * b.norm()


@pytest.mark.parametrize("dtype,sizes", [(torch.bfloat16, (1.0, 2.0 ** 12)), (torch.bfloat16, (2.0 ** 12, 1.0)), (torch.bfloat16, (2.0 ** -100, 2.0 ** 100)),
                                         (torch.bfloat16, (2.0 ** 100, 2.0 ** -100)), (torch.bfloat16, (2.0 ** 100,)), (torch.bfloat16, (2.0 ** -115,)),
                                         (torch.float16, (2.0 ** -18,)), (torch.float16, (2.0 ** -20, 2.0 ** 10))])
@pytest.mark.parametrize("hq,hk,head_dim,news", [(hq, hk, 128, news) for hq, hk, news in ROWS] + [(8, 2, 64, [2, 4])])
def test_keys_may_differ_in_size(backend, hq, hk, head_dim, news, dtype, sizes):
    """Pages of values of one size after pages of another."""
    cache = make_quantized(50, 16, hk, head_dim, dtype)
    batch, tokens = make_batch([500, 130], news, 16, 50, 2)
    for s in range(2):
        pages = batch.page_table[s][batch.page_table[s] >= 0].long()
        for size, part in zip(sizes, pages.chunk(len(sizes))):
            cache.v_steps[part] *= size
    q = torch.randn(tokens, hq, head_dim, generator=torch.Generator().manual_seed(5)).to(dtype).cuda()
    batch = of_the_step(batch, news)
    near(backend, q, cache, batch, head_dim ** -0.5, vanishes=vanishing(cache, hq, 500))


@pytest.mark.parametrize("hq,hk,head_dim,news", [(hq, hk, 128, news) for hq, hk, news in ROWS] + [(8, 2, 64, [2, 4]), (32, 2, 64, [2, 1])])
def test_runs_of_a_few_sequences_repeat(backend, hq, hk, head_dim, news):
    """A cluster's CTAs put their warps' states together in the place of the first warp's, which all lanes read before one writes it."""
    cache = make_quantized(50, 16, hk, head_dim, torch.float16)
    wide = PagedCache(*(quant.values(codes, steps).half() for codes, steps in (cache._tensors[:2], cache._tensors[2:])))
    batch, tokens = make_batch([500, 130], news, 16, 50, 2)
    batch = of_the_step(batch, news)
    q = torch.randn(tokens, hq, head_dim, generator=torch.Generator().manual_seed(5)).half().cuda()
    want = near(backend, q, cache, batch, head_dim ** -0.5), backend.attention_paged(q, wide, batch, head_dim ** -0.5)
    for _ in range(200):
        assert torch.equal(backend.attention_paged(q, cache, batch, head_dim ** -0.5), want[0])
        assert torch.equal(backend.attention_paged(q, wide, batch, head_dim ** -0.5), want[1])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hk,head_dim,news", [(8, 2, 128, [1, 1]), (8, 2, 128, [3, 4]), (8, 8, 128, [8, 5]), (8, 2, 64, [8, 3])])
@pytest.mark.parametrize("k_size,v_size,shift", [(30.0, 1.0, 0.0), (1e-3, 1e-4, 0.0), (1.0, 1000.0, 0.0), (1.0, 1.0, 40.0), (0.05, 1e-4, 3.0)])
def test_magnitudes(backend, dtype, hq, hk, head_dim, news, k_size, v_size, shift):
    cache = make_quantized(50, 16, hk, head_dim, dtype, shift=shift)
    cache.k_steps.mul_(k_size)
    cache.v_steps.mul_(v_size)
    cache.v_steps[7:20].mul_(2.0 ** -6)
    batch, tokens = make_batch([500, 130], news, 16, 50, 2)
    q = torch.randn(tokens, hq, head_dim, generator=torch.Generator().manual_seed(5)).to(dtype).cuda()
    near(backend, q, cache, of_the_step(batch, news), 128 ** -0.5, vanishes=vanishing(cache, hq, 500))
    near(backend, q * 2.0 ** -8, cache, of_the_step(batch, news), 1.0, vanishes=vanishing(cache, hq, 500))


@pytest.mark.parametrize("layout", ["rows", "heads", "joined"])
@pytest.mark.parametrize("size", [1, 5, 16, 48, 1000])
@pytest.mark.parametrize("head_dim,lengths,news", [(128, [300, 1000, 1], [1, 1, 1]), (128, [300, 1000, 2], [3, 4, 2]), (64, [300, 1000, 8], [8, 1, 8])])
def test_layouts_and_page_sizes(backend, layout, size, head_dim, lengths, news):
    pages = sum(-(-n // size) for n in lengths) + 2
    cache = make_quantized(pages, size, 2, head_dim, torch.float16, layout)
    batch, tokens = make_batch(lengths, news, size, pages, 2)
    spoil_unused(cache, batch)
    q = torch.randn(tokens, 8, head_dim, generator=torch.Generator().manual_seed(5)).half().cuda()
    # "joined" rows of 72 and 36 bytes begin off 16: the general kernel, which rounds nothing
    near(backend, q, cache, of_the_step(batch, news), head_dim ** -0.5, kernel="general" if layout == "joined" else "rows")


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("hq,hk,head_dim,news", [(8, 2, 128, [1, 0, 4, 2]), (8, 8, 128, [16, 1, 0, 9]), (16, 2, 64, [4, 1, 0, 3])])
def test_rows_in_front_of_their_keys(backend, causal, hq, hk, head_dim, news):
    lengths = [700, 3, 2, 1]                         # fewer keys than new tokens among them
    cache = make_quantized(60, 16, hk, head_dim, torch.bfloat16)
    batch, tokens = make_batch(lengths, news, 16, 60, 2)
    spoil_unused(cache, batch)
    q = torch.randn(tokens, hq, head_dim, generator=torch.Generator().manual_seed(5)).bfloat16().cuda()
    for zero in (False, True):
        near(backend, q, cache, of_the_step(batch, news), head_dim ** -0.5, causal=causal, zero_fully_masked=zero)


@pytest.mark.parametrize("hq,hk,head_dim", [(32, 8, 128), (16, 4, 64), (8, 8, 128)])
@pytest.mark.parametrize("news", [[1] * 11 + [90], [1, 0, 40, 1, 1, 0, 0, 1, 1, 1, 1, 60]])
def test_single_tokens_beside_chunks_keep_their_digits(backend, hq, hk, head_dim, news):
    lengths = [n + 137 * i for i, n in enumerate(news)]
    pages = sum(-(-n // 16) for n in lengths) + 3
    cache = make_quantized(pages, 16, hk, head_dim, torch.bfloat16, seed=6)
    batch, tokens = make_batch(lengths, news, 16, pages, 2)
    q = torch.randn(tokens, hq, head_dim, generator=torch.Generator().manual_seed(3)).bfloat16().cuda()
    near(backend, q, cache, of_the_step(batch, news), head_dim ** -0.5, kernel=[name for n in news for name in (["rows"] if n == 1 else ["chunk"] * n)])


def test_a_cache_beyond_32_bit_offsets(backend):
    pages, size, hk, d = 40000, 128, 8, 128
    cache = QuantizedCache.zeros(pages, size, hk, d)
    picked = torch.tensor([[39999, 3, 37000], [38888, 36500, 1]], dtype=torch.int32, device="cuda")
    for page in picked.flatten().tolist():
        for to, t in zip(cache._tensors, make_quantized(1, size, hk, d, torch.bfloat16, seed=page)._tensors):
            to[page] = t[0]
    for news in ([1, 1], [3, 2]):
        batch = PagedBatch(picked, torch.tensor([300, 384], dtype=torch.int32, device="cuda"), torch.tensor([0, news[0], sum(news)], dtype=torch.int32, device="cuda"),
                           max_query=max(news))
        near(backend, torch.randn(sum(news), 32, d, device="cuda").bfloat16(), cache, batch, 0.1)
