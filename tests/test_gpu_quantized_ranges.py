"""Attention over a cache in four bits at the ends of what its types hold: the few-rows kernel held to its own bound, that of scores
kept to f32 and of probabilities, weighed by the steps, in f16 (tests/quantized_reference.attention, "rows")."""
import pytest
import torch

from tests import quantized_reference as quant
from tests.test_gpu_quantized_cache import make_quantized
from tests.test_gpu_rope import make_batch
from vibe_compiler_b200.paged_cache import PagedBatch

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
    batch = PagedBatch(batch.page_table, batch.key_lengths, batch.query_starts, max_query=max(news))
    near(backend, q, cache, batch, scale)
