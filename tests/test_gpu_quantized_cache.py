"""A paged KV cache held in four bits: quantised writes, reading back, moved pages, and attention over the codes (bounds:
tests/quantized_reference.attention)."""
import copy

import pytest
import torch

from tests import paged_reference as ref
from tests import quantized_reference as quant
from tests.test_gpu_attention_paged import CASES
from tests.test_gpu_rope import make_batch, make_cache
from vibe_compiler_b200.backend import WB200Error
from vibe_compiler_b200.paged_cache import PagedBatch, PagedCache, PageTables, QuantizedCache, RotaryTable

pytestmark = pytest.mark.gpu


def make_quantized(pages, size, heads, head_dim, dtype, layout="heads", seed=1, shift=0):
    """Random rows in four bits. Layouts: rows of a head behind one another, heads of a row, codes and steps of a row side by side."""
    g = torch.Generator().manual_seed(seed)
    tensors = []
    for _ in range(2):
        codes, steps = quant.quantized((torch.randn(pages, size, heads, head_dim, generator=g) + shift).to(dtype))
        codes, steps = codes.cuda(), steps.cuda()
        if layout == "heads":
            codes, steps = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (codes, steps))
        elif layout == "joined":
            wide = codes.shape[3] + 4 * steps.shape[3]
            buffer = torch.zeros(pages, size, heads, wide, dtype=torch.uint8, device="cuda")
            buffer[..., :codes.shape[3]] = codes
            buffer[..., codes.shape[3]:] = steps.contiguous().view(torch.uint8).flatten(-2)
            codes = buffer[..., :codes.shape[3]]
            steps = buffer[..., codes.shape[3]:].view(dtype).unflatten(-1, (-1, 2))
        tensors += [codes, steps]
    return QuantizedCache(*tensors)


def spoil_unused(cache, batch):
    """Pairs that read back as NaN and infinity wherever no sequence has a key."""
    size = cache.page_size
    used = torch.zeros(cache.shape[:2], dtype=torch.bool)
    for row, n in zip(batch.page_table.cpu().tolist(), batch.key_lengths.tolist()):
        for j in range(n):
            used[row[j // size], j % size] = True
    used = used.cuda()
    cache.k_steps[~used] = float("nan")
    cache.v_steps[~used] = float("inf")
    cache.k_codes[~used] = 255
    cache.v_codes[~used] = 255


def agree(backend, q, cache, batch, scale, kernel="chunk", **options):
    lse = torch.full(q.shape[:2], 5.0, device="cuda")
    out = torch.full_like(q, 3.0)
    backend.attention_paged(q, cache, batch, scale, lse=lse, out=out, **options)
    backend.poll()
    want, want_lse, bound, bound_lse = quant.attention(q, cache, batch, scale, kernel=kernel, **options)
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


def check(got, want, norms, magnitude):
    """The bound of tests/test_gpu_rope.py for rows that hold subnormal numbers of the type too: their steps are all of one size, that
    of the smallest normal number's, eps * smallest_normal, so a rounding is off by half of that where unit * |want| says less."""
    info = torch.finfo(got.dtype)
    unit, floor = info.eps / 2, info.eps / 2 * info.smallest_normal
    bound = 8 * 2.0 ** -24 * abs(magnitude) * norms * (1 + unit) + (unit * want.abs()).clamp(min=floor)
    error = (got.cpu().double() - want).abs()
    assert bool((error <= bound).all()), ((error - bound).max().item(), got.dtype)


APPENDS = [([5, 1, 0, 40], [1, 1, 0, 1], 16, 8, 2, 128, 128), ([130, 33, 64], [130, 7, 64], 32, 7, 1, 64, 48), ([9, 10], [9, 3], 3, 2, 2, 24, 8),
           ([70], [70], 16, 0, 3, 256, 256), ([50, 3], [20, 3], 5, 3, 3, 80, 0), ([33], [33], 16, 4, 4, 200, 100), ([40], [31], 16, 2, 1, 8, 6)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("layout", ["rows", "heads", "joined"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("lengths,news,size,hq,hk,head_dim,rotary_dim", APPENDS)
def test_append_quantises_the_rows_of_its_tokens_only(backend, dtype, layout, lengths, news, size, hq, hk, head_dim, rotary_dim, interleaved):
    pages = sum(-(-n // size) for n in lengths) + 3
    cache = make_quantized(pages, size, hk, head_dim, dtype, layout)
    batch, tokens = make_batch(lengths, news, size, pages, 2, spare_rows=2)
    want = [t.cpu().clone() for t in cache._tensors]
    qkv = torch.randn(tokens, (hq + 2 * hk) * head_dim, generator=torch.Generator().manual_seed(3)).to(dtype)
    qkv[0] *= 1e-4                                   # small steps, in f16 among them subnormal ones
    qkv[-3] *= 100.0
    qkv = qkv.cuda()
    table = RotaryTable(rotary_dim, theta=1000.0, scaling="linear", factor=2.0, magnitude=1.25)
    out = torch.full((tokens, hq, head_dim), 7.0, dtype=dtype, device="cuda")
    backend.rope_append(qkv, cache, batch, table, q_heads=hq, interleaved=interleaved, out=out)
    backend.poll()
    rows = qkv.view(tokens, hq + 2 * hk, head_dim)
    at, page_table, turned_rows, places = 0, batch.page_table.cpu(), [], []
    for s, (length, n) in enumerate(zip(lengths, news)):
        for i in range(n):
            position = length - n + i
            token = rows[at:at + 1, :hq + hk]
            turned, norms = ref.rotated(token, torch.tensor([position]), table, interleaved)[0], ref.pair_norms(token, table, interleaved)[0]
            if hq:
                check(out[at], turned[:hq], norms[:hq], 1.25)
            k = turned[hq:].float().to(dtype)        # rounded as the format is defined: f64, f32, the type
            k[..., rotary_dim:] = rows[at, hq:hq + hk, rotary_dim:].cpu()
            turned_rows.append(k)
            places.append((int(page_table[s, position // size]), position % size))
            at += 1
    page, row = torch.tensor(places).T
    want[0][page, row], want[1][page, row] = quant.quantized(torch.stack(turned_rows))
    want[2][page, row], want[3][page, row] = quant.quantized(rows[:at, hq + hk:])
    for got, exact in zip(cache._tensors, want):
        assert torch.equal(got.cpu(), exact)
    assert bool((out[at:] == 7.0).all())             # tokens behind the last sequence
    # read back: the format's values, rounded once
    k, v = (torch.full((tokens, hk, head_dim), 7.0, dtype=dtype, device="cuda") for _ in range(2))
    backend.cache_read(cache, batch, tokens, out=(k, v))
    backend.poll()
    for got, codes, steps in ((k, want[0], want[1]), (v, want[2], want[3])):
        assert torch.equal(got[:at].cpu(), quant.values(codes[page, row], steps[page, row]).float().to(dtype))
        assert bool((got[at:] == 7.0).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_elements_are_within_half_a_step(backend, dtype):
    g = torch.Generator().manual_seed(5)
    x = torch.randn(200, 3, 128, generator=g) * torch.exp(6 * torch.randn(200, 3, 1, generator=g)) + 5 * torch.randn(200, 3, 1, generator=g)
    if dtype == torch.float16:
        x = x.clamp(-60000, 60000)
    qkv = x.to(dtype).cuda()
    cache, batch = QuantizedCache.zeros(16, 16, 1, 128, dtype), make_batch([200], [200], 16, 16, 2)[0]
    backend.rope_append(qkv.view(200, -1), cache, batch, None, q_heads=1)
    at = torch.arange(200, device="cuda")
    page, row = batch.page_table[0].long()[at // 16], at % 16
    for codes, steps, rows in ((cache.k_codes, cache.k_steps, qkv[:, 1:2]), (cache.v_codes, cache.v_steps, qkv[:, 2:3])):
        got, step = quant.values(codes[page, row], steps[page, row]), steps[page, row].double()[..., 0].repeat_interleave(64, -1)
        # half a step, and the f32 difference's and quotient's roundings
        assert bool(((got - rows.double()).abs() <= step * (0.5 + 2.0 ** -19)).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_rows_at_the_ends_of_the_type_stay_in_it(backend, dtype):
    """Fifteen steps, rounded up, would lead beyond the type's largest number: the step is rounded down."""
    largest = torch.finfo(dtype).max
    low = 0.0 if dtype == torch.bfloat16 else -largest                          # bf16: a wider range leaves f32
    rows = torch.stack([low * scale + (largest - low) * scale * torch.rand(128, generator=torch.Generator().manual_seed(i)) for i, scale in enumerate([1.0] * 6 + [0.99, 0.5])])
    rows[:, 3], rows[:, 5] = torch.tensor([low] * 6 + [low * 0.99, low * 0.5]), torch.tensor([largest] * 6 + [largest * 0.99, largest * 0.5])
    rows[:, 64], rows[:, 127] = rows[:, 3], rows[:, 5]
    qkv = torch.stack((rows, rows.flip(0), rows), 1).to(dtype).cuda()
    cache, batch = QuantizedCache.zeros(2, 16, 1, 128, dtype), make_batch([8], [8], 16, 2, 2)[0]
    backend.rope_append(qkv.view(8, -1), cache, batch, None, q_heads=1)
    for got, x in zip(backend.cache_read(cache, batch, 8), (qkv[:, 1:2], qkv[:, 2:])):
        codes, steps = quant.quantized(x)
        assert torch.equal(got.cpu(), quant.values(codes, steps).float().to(dtype)) and bool(got.isfinite().all())
        step = steps.double()[..., 0].repeat_interleave(64, -1)
        # half a step, 15 units in the step's last place where it was rounded down, and the result's rounding
        eps = torch.finfo(dtype).eps
        assert bool(((got.cpu().double() - x.cpu().double()).abs() <= step * (0.5 + 15 * eps + 2.0 ** -19) + x.cpu().double().abs() * eps).all())
    backend.poll()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_groups_without_a_range_and_with_odd_values(backend, dtype):
    """Equal elements, zeros of both signs, the type's largest values, infinities and NaN: what they read back as."""
    largest, tiny = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal / 2 ** (7 if dtype == torch.bfloat16 else 10)
    rows = torch.zeros(8, 128)
    rows[0], rows[1, ::2], rows[2, 3] = 3.0, -0.0, float("inf")
    rows[3, 70] = float("nan")
    rows[4, 0], rows[4, 1] = largest / 4, -largest / 4
    rows[5, 5], rows[5, 6] = tiny, -tiny
    rows[6, 64:], rows[6, 100] = 100.0, 100.5
    rows[7, 9] = -float("inf")
    qkv = torch.stack((rows, rows.flip(0), rows), 1).to(dtype).cuda()
    cache, batch = QuantizedCache.zeros(2, 16, 1, 128, dtype), make_batch([8], [8], 16, 2, 2)[0]
    backend.rope_append(qkv.view(8, -1), cache, batch, None, q_heads=1)
    k, v = backend.cache_read(cache, batch, 8)
    backend.poll()
    for got, x in ((k, qkv[:, 1:2]), (v, qkv[:, 2:])):
        codes, steps = quant.quantized(x)
        want = quant.values(codes, steps).float().to(dtype)
        assert torch.equal(got.cpu().isnan(), want.isnan()) and torch.equal(got.cpu().nan_to_num(), want.nan_to_num())
    v = v[:, 0].cpu().float()
    assert bool((v[0] == 3.0).all()) and bool((v[1] == 0.0).all())
    assert bool(v[2, :64].isnan().all()) and bool((v[2, 64:] == 0.0).all()) and bool(v[3, 64:].isnan().all()) and bool((v[3, :64] == 0.0).all())
    assert v[4, 1] == rows[4, 1] and abs(v[4, 0] / rows[4, 0] - 1) <= 2.0 ** -6
    assert bool((v[5].abs() <= tiny).all()) and v[6, 64] == 100.0 and v[6, 100] == 100.5 and bool(v[7, :64].isnan().all())


def test_append_with_positions_of_its_own(backend):
    cache = make_quantized(8, 16, 2, 64, torch.bfloat16)
    batch, tokens = make_batch([20, 30], [3, 2], 16, 8, 2)
    qkv = torch.randn(tokens, 8 * 64, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    table, rows = RotaryTable(64), qkv.view(tokens, 8, 64)
    for dtype in (torch.int32, torch.int64):
        positions = torch.tensor([100, 7, 0, 5, 999], dtype=dtype, device="cuda")
        q = backend.rope_append(qkv, cache, batch, table, q_heads=4, positions=positions)
        assert torch.equal(q, backend.rope(rows[:, :4], positions, table))
        want = ref.rotated(rows[:, 4:6], positions, table).float().bfloat16()
        page, row = batch.page_table[0].long()[1], torch.arange(1, 4)          # keys 17 to 19
        assert all(torch.equal(a.cpu(), b) for a, b in zip((cache.k_codes[page, row], cache.k_steps[page, row]), quant.quantized(want[:3])))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind", ["16-bit rows", "16-bit heads", "16-bit odd", "four bits", "four bits, rows", "four bits, joined"])
@pytest.mark.parametrize("lengths,news,size,hk,head_dim", [
    ([5, 1, 0, 40], [5, 1, 0, 40], 16, 2, 128), ([130, 33, 64], [130, 7, 0], 32, 1, 64), ([9, 10], [9, 3], 3, 2, 24), ([3000, 700], [3000, 699], 64, 8, 128)])
def test_read_gives_the_rows_of_the_batch(backend, dtype, kind, lengths, news, size, hk, head_dim):
    pages = sum(-(-n // size) for n in lengths) + 3
    if kind.startswith("16"):
        cache = make_cache(pages, size, hk, head_dim, dtype, "heads" if kind.endswith("heads") else "rows", 1)
        if kind.endswith("odd"):                     # rows that begin off 16 bytes
            cache = PagedCache(*(torch.cat((t.flatten()[:1], t.flatten()))[1:].view(t.shape) for t in (cache.k, cache.v)))
        stored = cache.k.double(), cache.v.double()
    else:
        cache = make_quantized(pages, size, hk, head_dim, dtype, kind[11:] or "heads")
        stored = quant.values(cache.k_codes, cache.k_steps), quant.values(cache.v_codes, cache.v_steps)
    batch, tokens = make_batch(lengths, news, size, pages, 2, spare_rows=3)
    outs = [torch.full((tokens, hk, head_dim), 5.0, dtype=dtype, device="cuda"), torch.full((hk, tokens, head_dim + 1), 5.0, dtype=dtype, device="cuda")]
    views = outs[0], outs[1].transpose(0, 1)[..., :head_dim]                   # V to rows off 16 bytes, heads outside tokens
    assert backend.cache_read(cache, batch, tokens, out=views)[0] is views[0]
    plain = backend.cache_read(cache, batch, tokens)
    backend.poll()
    at = 0
    for s, (length, n) in enumerate(zip(lengths, news)):
        for got, other, store in zip(views, plain, stored):
            want = ref.gathered(store, batch.page_table[s], length, size)[length - n:].float().to(dtype)
            assert torch.equal(got[at:at + n], want) and torch.equal(other[at:at + n], want)
        at += n
    assert bool((outs[0][at:] == 5.0).all()) and bool((outs[1][:, at:] == 5.0).all()) and bool((outs[1][..., head_dim:] == 5.0).all())


@pytest.mark.parametrize("fault", ["page too large", "page negative", "length beyond the table", "more tokens than keys", "a range ends behind the rows"])
def test_writes_and_reads_leave_out_rows_without_a_place(backend, fault):
    cache = make_quantized(8, 16, 2, 64, torch.float16)
    batch, tokens = make_batch([20, 30], [3, 2], 16, 8, 2)
    before = [t.clone() for t in cache._tensors]
    first = batch.page_table[0].long().tolist()
    if fault.startswith("page"):
        batch.page_table[1, 1] = 8 if fault == "page too large" else -1
    elif fault.startswith("a range"):
        batch.query_starts[2] = tokens + 40
    else:
        batch.key_lengths[1] = 1000 if fault.startswith("length") else 1
    qkv = torch.randn(tokens, 8 * 64, device="cuda").half()
    backend.rope_append(qkv, cache, batch, RotaryTable(64), q_heads=4)
    with pytest.raises(WB200Error, match="left out"):
        backend.poll()
    backend.poll()                                    # reported once
    allowed = set(first[:2]) | ({int(batch.page_table[1, 0])} if fault.startswith("more") else set())
    for now, was in zip(cache._tensors, before):
        changed = (now != was).flatten(1).any(1).nonzero().flatten().tolist()
        assert set(changed) <= allowed and first[1] in changed
        assert torch.equal(now[first[0], :16], was[first[0], :16])             # keys 17 to 19 lie in the second page
    k, v = (torch.full((tokens, 2, 64), 5.0, dtype=torch.float16, device="cuda") for _ in range(2))
    backend.cache_read(cache, batch, tokens, out=(k, v))
    with pytest.raises(WB200Error, match="left out"):
        backend.poll()
    at = torch.arange(17, 20, device="cuda")
    page = batch.page_table[0].long()[at // 16]
    assert torch.equal(v[:3], quant.values(cache.v_codes[page, at % 16], cache.v_steps[page, at % 16]).float().half())
    left_out = slice(3, 4 if fault.startswith("more") else 5)                  # of two tokens and one key, the second has a place
    assert bool((v[left_out] == 5.0).all()) and bool((k[left_out] == 5.0).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lengths,news,size,hq,hk,head_dim", CASES)
def test_attention_matches_float64(backend, dtype, causal, lengths, news, size, hq, hk, head_dim):
    pages = sum(-(-n // size) for n in lengths) + 3
    cache = make_quantized(pages, size, hk, head_dim, dtype)
    batch, tokens = make_batch(lengths, news, size, pages, 2, spare_rows=3)
    spoil_unused(cache, batch)
    q = torch.randn(tokens, hq, head_dim, generator=torch.Generator().manual_seed(3)).to(dtype).cuda()
    wide, _ = make_batch(lengths, news, size, pages, 2, width=65536 // size + 2)     # room for longer sequences
    for max_query, table in ((0, batch.page_table), (1, batch.page_table), (max(news), batch.page_table), (1, wide.page_table), (0, wide.page_table)):
        hinted = PagedBatch(table, batch.key_lengths, batch.query_starts, max_query=max_query)      # a hint: right, wrong or missing
        agree(backend, q, cache, hinted, head_dim ** -0.5, causal=causal, zero_fully_masked=max_query == 1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("size,hq,hk,head_dim", [(16, 32, 8, 128), (32, 8, 8, 128), (48, 28, 4, 128), (5, 16, 1, 128), (64, 16, 4, 64), (7, 8, 8, 64), (16, 9, 3, 80)])
@pytest.mark.parametrize("lengths", [[700, 64, 65, 2000, 0, 1], [33], [9000, 129, 31]])
def test_few_tokens_take_scores_to_f32(backend, dtype, size, hq, hk, head_dim, lengths):
    """Without rounded keys: scores to f32's bound, in the log-sum-exp too, and probabilities to f16's (kept in f32 at other head
    dimensions), whatever the type."""
    pages = sum(-(-n // size) for n in lengths) + 3
    cache = make_quantized(pages, size, hk, head_dim, dtype, seed=4)
    for n in range(1, max(1, 16 * hk // hq) + 1):
        batch, tokens = make_batch([x + n for x in lengths], [n] * len(lengths), size, pages + len(lengths) * (1 + n // size), 2)
        batch.page_table.clamp_(max=pages - 1)       # sequences may share pages that are only read
        q = torch.randn(tokens, hq, head_dim, generator=torch.Generator().manual_seed(n)).to(dtype).cuda()
        q[0] *= 2.0 ** -12                           # a row of small scores beside others
        hinted = PagedBatch(batch.page_table, batch.key_lengths, batch.query_starts, max_query=n)
        agree(backend, q, cache, hinted, head_dim ** -0.5, kernel="rows" if head_dim != 80 else "general")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hk,head_dim", [(32, 8, 128), (8, 8, 128), (28, 4, 128), (16, 1, 128), (16, 4, 64)])
def test_means_of_many_values_keep_their_digits(backend, dtype, hq, hk, head_dim):
    """Values around zero, 30 thousand to a row: the result is 1/100 of a value. In the 2-norm, relative to the result, with u half a
    step of the type:
      p'       off by 2^-11 at most, uniformly and apart from one another: 2^-11 / sqrt(3) of (code - 8) step, which is a value's size
      sums     a product's f32 sums are cut off at 2^-23 of 16 keys' 136 p' at most: 136 step 2^-23 <= 8e-6 (steps up to 0.5), and the
               result is 1 / sqrt(sum p^2) >= 1/200 of a value: 1.6e-3
      result   u / sqrt(3)"""
    cache = make_quantized(500, 64, hk, head_dim, dtype, seed=8)
    batch, tokens = make_batch([30000, 20000 // 20], [1, 1], 64, 500, 2)
    q = torch.randn(tokens, hq, head_dim, generator=torch.Generator().manual_seed(3)).to(dtype).cuda()
    got = backend.attention_paged(q, cache, batch, head_dim ** -0.5).double()
    backend.poll()
    want = quant.attention(q, cache, batch, head_dim ** -0.5)[0]
    u = torch.finfo(dtype).eps / 2
    for row in range(tokens):
        assert (got[row] - want[row]).norm() <= (2.0 ** -11 / 3 ** 0.5 + 1.6e-3 + u / 3 ** 0.5) * want[row].norm()


@pytest.mark.parametrize("layout", ["rows", "heads", "joined"])
@pytest.mark.parametrize("lengths,news", [([300, 1000], [1, 1]), ([300, 1000], [3, 4]), ([300, 1000], [200, 150])])
def test_layouts_and_strides(backend, layout, lengths, news):
    size, hq, hk, d = 32, 8, 2, 128
    cache = make_quantized(50, size, hk, d, torch.bfloat16, layout)
    batch, tokens = make_batch(lengths, news, size, 50, 2)
    fused = torch.randn(tokens, hq + 2 * hk, d, generator=torch.Generator().manual_seed(5)).bfloat16().cuda()
    want = agree(backend, fused[:, :hq], cache, batch, 0.1)
    assert torch.equal(backend.attention_paged(fused[:, :hq].contiguous(), cache, batch, 0.1), want)
    out = torch.empty(hq, tokens, d, dtype=torch.bfloat16, device="cuda").transpose(0, 1)
    backend.attention_paged(fused[:, :hq], cache, batch, 0.1, out=out)
    backend.poll()
    assert torch.equal(out, want)
    odd = torch.zeros(fused[:, :hq].numel() + 3, dtype=torch.bfloat16, device="cuda")[3:].view(tokens, hq, d)      # off 16 bytes
    odd.copy_(fused[:, :hq])
    agree(backend, odd, cache, batch, 0.1)
    heads_outside = fused[:, :hq].transpose(0, 1).contiguous().transpose(0, 1)
    agree(backend, heads_outside, cache, batch, 0.1)


@pytest.mark.parametrize("lengths,news", [([90, 40], [1, 1]), ([90, 40, 10], [60, 50, 30])])
def test_rows_without_keys(backend, lengths, news):
    # more new tokens than keys: the first ones stand in front of key 0
    lengths = [n // 2 for n in lengths]
    cache = make_quantized(20, 16, 2, 128, torch.float16)
    batch, tokens = make_batch(lengths, news, 16, 20, 2)
    spoil_unused(cache, batch)
    q = torch.randn(tokens, 8, 128, device="cuda").half()
    for zero in (False, True):
        agree(backend, q, cache, batch, 0.1, zero_fully_masked=zero)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("news", [[1, 1], [5, 3], [40, 1]])
@pytest.mark.parametrize("k_size,v_size,shift", [(30.0, 1.0, 0.0), (1e-3, 1e-4, 0.0), (1.0, 1000.0, 0.0), (1.0, 1.0, 40.0), (0.05, 1e-6, 3.0)])
def test_magnitudes(backend, dtype, news, k_size, v_size, shift):
    """Large and tiny scores and values, and rows far from zero: the products' scales and their cancellation."""
    cache = make_quantized(50, 16, 2, 128, dtype, shift=shift)
    if dtype == torch.float16 and v_size < 1e-5:
        v_size = 1e-4                                # steps stay normal numbers
    cache.k_steps.mul_(k_size)
    cache.v_steps.mul_(v_size)
    cache.v_steps[7:20].mul_(2.0 ** -6)              # and pages of different size in one row
    batch, tokens = make_batch([500, 130], news, 16, 50, 2)
    q = torch.randn(tokens, 8, 128, generator=torch.Generator().manual_seed(5)).to(dtype).cuda()
    agree(backend, q, cache, batch, 128 ** -0.5)
    agree(backend, q * 2.0 ** -8, cache, batch, 1.0)


@pytest.mark.parametrize("news", [[1, 1, 1], [80, 70, 3]])
def test_a_key_that_is_not_a_number_reaches_its_own_sequence_only(backend, news):
    cache = make_quantized(40, 16, 2, 128, torch.bfloat16)
    batch, tokens = make_batch([200, 150, 90], news, 16, 40, 2)
    q = torch.randn(tokens, 8, 128, device="cuda").bfloat16()
    want, _, bound, _ = quant.attention(q, cache, batch, 0.1)
    cache.k_steps[int(batch.page_table[1, 0]), 3, 1] = float("nan")            # seen by every row of sequence 1, KV head 1
    got = backend.attention_paged(q, cache, batch, 0.1).double()
    backend.poll()
    a, b = news[0], news[0] + news[1]
    assert bool(got[a:b, 4:].isnan().all())
    got[a:b, 4:], want[a:b, 4:] = 0.0, 0.0
    assert bool(((got - want).abs() <= bound).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("news,hq", [([1, 1], 8), ([1, 1], 16), ([8, 5], 4), ([70, 33], 8)])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_a_value_that_is_not_a_number_stays_in_its_group(backend, dtype, news, hq, value):
    cache = make_quantized(40, 16, 2, 128, dtype)
    batch, tokens = make_batch([200, 150], news, 16, 40, 2)
    q = torch.randn(tokens, hq, 128, generator=torch.Generator().manual_seed(3)).to(dtype).cuda()
    want, _, bound, _ = quant.attention(q, cache, batch, 0.1)
    cache.v_steps[int(batch.page_table[1, 0]), 3, 1, 0] = value                # seen by every row of sequence 1, KV head 1
    got = backend.attention_paged(q, cache, batch, 0.1).double()
    backend.poll()
    own = got[news[0]:, hq // 2:, :64]
    assert bool((~own.isfinite()).all())
    got[news[0]:, hq // 2:, :64], want[news[0]:, hq // 2:, :64] = 0.0, 0.0
    assert bool(((got - want).abs() <= bound).all())


def test_results_do_not_depend_on_where_the_pages_lie_or_on_the_run(backend):
    size, lengths = 16, [900, 5000, 33, 260]
    cache = make_quantized(420, size, 4, 128, torch.bfloat16)
    for news in ([1, 1, 1, 1], [2, 1, 3, 2], [100, 40, 33, 1]):
        batch, tokens = make_batch(lengths, news, size, 420, 2)
        q = torch.randn(tokens, 28, 128, device="cuda").bfloat16()
        want = backend.attention_paged(q, cache, batch, 0.09)
        for _ in range(5):
            assert torch.equal(backend.attention_paged(q, cache, batch, 0.09), want)
        order = torch.randperm(420, device="cuda")
        moved = QuantizedCache(*(torch.empty_like(t) for t in cache._tensors))
        for to, t in zip(moved._tensors, cache._tensors):
            to[order] = t
        table = torch.where(batch.page_table >= 0, order[batch.page_table.clamp(min=0).long()].int(), batch.page_table)
        assert torch.equal(backend.attention_paged(q, moved, PagedBatch(table, batch.key_lengths, batch.query_starts), 0.09), want)


@pytest.mark.parametrize("news", [[1, 1], [3, 2], [80, 70]])
@pytest.mark.parametrize("fault", ["page too large", "page negative", "length beyond the table", "tokens beyond the rows"])
def test_bad_device_data_is_left_out_and_reported(backend, news, fault):
    cache = make_quantized(30, 16, 2, 128, torch.bfloat16)
    batch, tokens = make_batch([200, 150], news, 16, 30, 2)
    q = torch.randn(tokens, 8, 128, device="cuda").bfloat16()
    want, _, bound, _ = quant.attention(q, cache, batch, 0.1)
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


@pytest.mark.parametrize("news", [[1, 1, 1], [2, 4, 3], [200, 1, 64]])
def test_calls_on_two_streams_at_once(backend, news):
    cache = make_quantized(600, 16, 4, 128, torch.float16)
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


def test_captured_calls_follow_the_lengths_on_the_device(backend):
    size = 16
    cache = make_quantized(600, size, 4, 128, torch.bfloat16)
    long, tokens = make_batch([4000, 900, 2000], [1, 1, 1], size, 600, 2)
    qkv = torch.randn(tokens, 36 * 128, device="cuda").bfloat16()
    batch = PagedBatch(long.page_table.clone(), long.key_lengths.clone(), long.query_starts.clone(), max_query=1)
    table = RotaryTable(128)

    def step():
        q = backend.rope_append(qkv, cache, batch, table, q_heads=28)
        return (q, backend.attention_paged(q, cache, batch, 0.1), *backend.cache_read(cache, batch, tokens))
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for lengths in ([4000, 900, 2000], [17, 4000, 1], [3, 5, 3999]):
        batch.key_lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
        wide, _ = make_batch(lengths, [1, 1, 1], size, 600, 9, width=batch.page_table.shape[1])
        batch.page_table.copy_(wide.page_table)
        for _ in range(2):
            graph.replay()
        got = [t.clone() for t in outs]
        assert all(torch.equal(a, b) for a, b in zip(got, step()))
    backend.poll()


def test_more_sequences_than_a_block_stages(backend):
    count = 5000
    news = [0] * count
    news[17], news[4999], news[3000] = 40, 1, 9
    lengths = [0] * count
    lengths[17], lengths[4999], lengths[3000], lengths[4] = 70, 33, 9, 16
    cache = make_quantized(20, 16, 2, 128, torch.bfloat16)
    batch, tokens = make_batch(lengths, news, 16, 20, 2)
    agree(backend, torch.randn(tokens, 8, 128, device="cuda").bfloat16(), cache, batch, 0.1)
    few = PagedBatch(batch.page_table[:4000], batch.key_lengths[:4000].contiguous(), batch.query_starts[:4001].contiguous())
    agree(backend, torch.randn(tokens, 8, 128, device="cuda").bfloat16(), cache, few, 0.1)


@pytest.mark.parametrize("size", [1, 1000])
def test_pages_of_one_row_and_of_a_sequence(backend, size):
    lengths = [300, 41, 1]
    cache = make_quantized(sum(-(-n // size) for n in lengths) + 2, size, 2, 128, torch.float16)
    for news in ([1, 1, 1], [2, 4, 1], [70, 41, 1], [300, 0, 0]):
        batch, tokens = make_batch(lengths, news, size, cache.shape[0], 2)
        spoil_unused(cache, batch)
        q = torch.randn(tokens, 8, 128, generator=torch.Generator().manual_seed(3)).half().cuda()
        for max_query in (0, max(news)):
            agree(backend, q, cache, PagedBatch(batch.page_table, batch.key_lengths, batch.query_starts, max_query=max_query), 0.1)


def test_one_page_in_many_places(backend):
    # a sequence may list a page more than once: 40 thousand keys over three pages
    cache = make_quantized(3, 128, 2, 128, torch.bfloat16)
    table = torch.arange(320, dtype=torch.int32, device="cuda")[None, :] % 3
    for n in (1, 70):
        batch = PagedBatch(table, torch.tensor([40900], dtype=torch.int32, device="cuda"), torch.tensor([0, n], dtype=torch.int32, device="cuda"))
        agree(backend, torch.randn(n, 8, 128, device="cuda").bfloat16(), cache, batch, 0.1)


@pytest.mark.parametrize("hq,hk,head_dim", [(32, 8, 128), (16, 4, 64), (8, 8, 128), (18, 1, 128)])
@pytest.mark.parametrize("news", [[1] * 11 + [90], [1, 0, 40, 1, 1, 0, 0, 2, 1, 1, 1, 60], [70] + [0] * 11, [0] * 5 + [33, 2] + [0] * 5])
def test_single_tokens_beside_chunks(backend, news, hq, hk, head_dim):
    """Batches whose single tokens and chunks go to kernels of their own, by what the host knows: neither writes the other's rows."""
    lengths = [n + 37 * i for i, n in enumerate(news)]
    pages = sum(-(-n // 16) for n in lengths) + 3
    cache = make_quantized(pages, 16, hk, head_dim, torch.bfloat16, seed=6)
    batch, tokens = make_batch(lengths, news, 16, pages, 2, spare_rows=2)
    spoil_unused(cache, batch)
    q = torch.randn(tokens, hq, head_dim, generator=torch.Generator().manual_seed(3)).bfloat16().cuda()
    hinted = PagedBatch(batch.page_table, batch.key_lengths, batch.query_starts, max_query=max(news))
    out = agree(backend, q, cache, hinted, head_dim ** -0.5)
    assert torch.equal(backend.attention_paged(q, cache, hinted, head_dim ** -0.5)[:tokens - 2], out[:tokens - 2])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again = backend.attention_paged(q, cache, hinted, head_dim ** -0.5)
    graph.replay()
    assert torch.equal(again[:tokens - 2], out[:tokens - 2])
    backend.poll()


def test_empty_calls(backend):
    cache = make_quantized(4, 16, 2, 128, torch.bfloat16)
    batch, _ = make_batch([20, 0], [0, 0], 16, 4, 2)
    nothing = torch.empty(0, 8, 128, dtype=torch.bfloat16, device="cuda")
    assert backend.attention_paged(nothing, cache, batch, 0.1).shape == (0, 8, 128)
    assert backend.rope_append(nothing.new_empty(0, 12 * 128), cache, batch, None, q_heads=8).shape == (0, 8, 128)
    assert [t.shape for t in backend.cache_read(cache, batch, 0)] == [(0, 2, 128)] * 2
    untouched = torch.full((3, 8, 128), 2.0, dtype=torch.bfloat16, device="cuda")
    backend.attention_paged(torch.zeros_like(untouched), cache, batch, 0.1, out=untouched)
    backend.poll()
    assert bool((untouched == 2.0).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("layout", ["rows", "heads", "joined"])
@pytest.mark.parametrize("head_dim", [64, 128, 24, 256])
def test_pages_move_with_their_steps(backend, dtype, layout, head_dim):
    caches = [make_quantized(12, 16, 3, head_dim, dtype, layout, seed=s) for s in (1, 2)]
    before = [[t.clone() for t in c._tensors] for c in caches]
    backend.pages_copy(caches, torch.tensor([3, -1, 7, 0], dtype=torch.int32, device="cuda"), torch.tensor([9, 4, 1, 11], dtype=torch.int32, device="cuda"))
    backend.poll()
    for cache, was in zip(caches, before):
        for now, then in zip(cache._tensors, was):
            then[9], then[1], then[11] = then[3].clone(), then[7].clone(), then[0].clone()
            assert torch.equal(now, then)
    with pytest.raises(ValueError, match="one kind"):
        backend.pages_copy([caches[0], make_cache(12, 16, 3, 64, dtype, "rows", 1)], *[torch.zeros(1, dtype=torch.int32, device="cuda")] * 2)


def test_a_cache_beyond_32_bit_offsets(backend):
    pages, size, hk, d = 40000, 128, 8, 128          # 2.6e9 bytes of codes each of K and V
    cache = QuantizedCache.zeros(pages, size, hk, d)
    picked = torch.tensor([[39999, 3, 37000], [38888, 36500, 1]], dtype=torch.int32, device="cuda")
    for page in picked.flatten().tolist():
        for to, t in zip(cache._tensors, make_quantized(1, size, hk, d, torch.bfloat16, seed=page)._tensors):
            to[page] = t[0]
    for news in ([1, 1], [3, 2], [100, 70]):
        tokens = sum(news)
        batch = PagedBatch(picked, torch.tensor([300, 384], dtype=torch.int32, device="cuda"), torch.tensor([0, news[0], tokens], dtype=torch.int32, device="cuda"))
        agree(backend, torch.randn(tokens, 32, d, device="cuda").bfloat16(), cache, batch, 0.1)
        qkv = torch.randn(tokens, (32 + 2 * hk) * d, device="cuda").bfloat16()
        backend.rope_append(qkv, cache, batch, None, q_heads=32)
        _, v = backend.cache_read(cache, batch, tokens)
        assert torch.equal(v.cpu(), quant.values(*quant.quantized(qkv.view(-1, 48, d)[:, 40:])).float().bfloat16())
    tables = torch.tensor([39999, 37000], dtype=torch.int32, device="cuda"), torch.tensor([5, 39998], dtype=torch.int32, device="cuda")
    backend.pages_copy(cache, *tables)
    assert torch.equal(cache.k_codes[5], cache.k_codes[39999]) and torch.equal(cache.v_steps[39998], cache.v_steps[37000])
    backend.poll()


def test_handles_follow_their_tensors(backend):
    cache, other = (make_quantized(8, 16, 2, 64, torch.bfloat16, seed=s) for s in (1, 2))
    batch, tokens = make_batch([20, 30], [3, 2], 16, 8, 2)
    copied = copy.deepcopy(cache)
    before = backend.cache_read(cache, batch, tokens)
    cache.v_codes.zero_()
    assert torch.equal(backend.cache_read(copied, batch, tokens)[1], before[1])
    for name in ("k_codes", "k_steps", "v_codes", "v_steps"):
        setattr(cache, name, getattr(other, name))
    assert all(torch.equal(a, b) for a, b in zip(backend.cache_read(cache, batch, tokens), backend.cache_read(other, batch, tokens)))


class CheckedBackend:
    """The backend, each of whose calls on a quantised cache is compared with the format and with attention in 64 bits."""

    def __init__(self, backend):
        self._backend, self.steps = backend, 0

    def __getattr__(self, name):
        return getattr(self._backend, name)

    def rope_append(self, qkv, cache, batch, table, *, q_heads):
        q = self._backend.rope_append(qkv, cache, batch, table, q_heads=q_heads)
        tokens, hk, d = qkv.shape[0], cache.shape[2], cache.shape[3]
        rows = qkv.view(tokens, -1, d)
        starts, lengths = batch.query_starts.tolist(), batch.key_lengths.tolist()
        positions = torch.cat([torch.arange(n - (b - a), n) for a, b, n in zip(starts, starts[1:], lengths)])
        wants = ref.rotated(rows[:, q_heads:q_heads + hk], positions, table).float().to(cache.dtype), rows[:, q_heads + hk:]
        for got, want in zip(self._backend.cache_read(cache, batch, tokens), wants):
            assert torch.equal(got.cpu(), quant.values(*quant.quantized(want)).float().to(cache.dtype))
        return q

    def attention_paged(self, q, cache, batch, scale, out=None):
        self._backend.attention_paged(q, cache, batch, scale, out=out)
        want, _, bound, _ = quant.attention(q, cache, batch, scale)
        assert bool(((out.double() - want).abs() <= bound).all())
        self.steps += 1
        return out


def test_a_serving_run(backend):
    """Prompts in pieces, decoding, drafted tokens, a fork, a freed sequence and moved pages through the decoder layer, every call on
    the quantised cache compared; the run stays near the one on a 16-bit cache."""
    from vibe_compiler_b200.decoder_layer import LayerConfig, ShardedDecoderLayer, random_weights
    cfg = LayerConfig(d_model=512, q_heads=8, kv_heads=2, head_dim=128, ffn=768)
    checked = CheckedBackend(backend)
    runs = []
    for be, make in ((checked, QuantizedCache.zeros), (backend, PagedCache.zeros)):
        layer = ShardedDecoderLayer(be, cfg, random_weights(cfg))
        tables, cache = PageTables(backend, 5, 24, 60, 16), make(60, 16, 2, 128)
        g = torch.Generator().manual_seed(11)
        done, outputs = [0] * 5, []

        def step(counts):
            for s, n in counts.items():
                done[s] += n
            assert int(tables.reserve(torch.tensor(done, dtype=torch.int32).cuda())) == 0
            starts = torch.tensor([0] + [counts.get(s, 0) for s in range(5)]).cumsum(0).to(torch.int32).cuda()
            x = torch.randn(sum(counts.values()), 512, generator=g).bfloat16().cuda()
            outputs.append(layer.forward_paged(x, cache, PagedBatch(tables.table, tables.lengths, starts, max_query=max(counts.values()))))

        step({0: 70, 1: 20, 3: 130})
        step({0: 1, 1: 1, 3: 33})
        assert int(tables.fork(torch.tensor([3], dtype=torch.int32).cuda(), torch.tensor([4], dtype=torch.int32).cuda(), [cache])) == 0
        done[4] = done[3]
        for _ in range(4):
            step({0: 1, 1: 1, 3: 1, 4: 1})
        tables.free(torch.tensor([1], dtype=torch.int32).cuda())
        done[1] = 0
        tables.compact([cache])
        for _ in range(3):
            step({0: 2, 3: 1, 4: 3})
        backend.poll()
        runs.append(torch.cat(outputs).double())
    assert checked.steps == 9
    # The residual path carries most of the output; a step of 1/15 of the range of 64 elements is what the caches differ by.
    assert (runs[0] - runs[1]).norm() <= 0.1 * runs[1].norm()
