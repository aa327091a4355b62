"""Rotary positions and the writes of new rows into a paged cache, against float64.

Bounds: sine and cosine are off by a few units of 2^-24 (angle remainder, sincospi, magnitude), the products and their sum by
one each, so an element is off by at most 8 * 2^-24 times magnitude * (|u| + |w|) of its pair, plus half a step of the type."""
import math

import pytest
import torch

from tests import paged_reference as ref
from vibe_compiler_b200.backend import WB200Error
from vibe_compiler_b200.paged_cache import PagedBatch, PagedCache, RotaryTable

pytestmark = pytest.mark.gpu


def check(got, want, norms, magnitude):
    unit = torch.finfo(got.dtype).eps / 2
    bound = 8 * 2.0 ** -24 * abs(magnitude) * norms * (1 + unit) + unit * want.abs()
    error = (got.cpu().double() - want).abs()
    assert bool((error <= bound).all()), ((error - bound).max().item(), got.dtype)


SHAPES = [(1, 1, 2, 2), (3, 5, 64, 64), (7, 3, 128, 96), (65, 40, 128, 128), (33, 2, 80, 40), (17, 3, 33, 10), (2000, 1, 256, 64), (5, 2, 96, 0)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,head_dim,rotary_dim", SHAPES)
def test_rope_matches_float64(backend, dtype, interleaved, tokens, heads, head_dim, rotary_dim):
    g = torch.Generator().manual_seed(tokens + heads)
    rows = torch.randn(tokens, heads + 1, head_dim, generator=g).to(dtype).cuda()
    x = rows[:, :heads]
    positions = torch.randint(0, 100000, (tokens,), generator=g, dtype=torch.int64 if tokens % 2 else torch.int32).cuda()
    table = RotaryTable(rotary_dim, theta=500000.0, scaling="yarn", factor=4.0, original_length=8192) if rotary_dim > 2 else RotaryTable(rotary_dim)
    for backward in (False, True):
        got = backend.rope(x, positions, table, interleaved=interleaved, backward=backward)
        check(got, ref.rotated(x, positions, table, interleaved, backward), ref.pair_norms(x, table, interleaved), table.magnitude)
        assert torch.equal(got[..., rotary_dim:], x[..., rotary_dim:])


@pytest.mark.parametrize("position", [0, -1, 12345678, 2 ** 31 - 1, -2 ** 40, 2 ** 52 + 1])
def test_far_positions_keep_their_angle(backend, position):
    # one pair at a time, its phase exact in integers: position * turns modulo 2^64
    table = RotaryTable(64, theta=10000.0)
    x = torch.zeros(1, 1, 64, device="cuda")
    x[..., :32] = 1.0
    got = backend.rope(x, torch.tensor([position], device="cuda"), table)[0, 0].cpu().double()
    for i in range(32):
        turns = (position * table._turns[i]) % 2 ** 64 / 2.0 ** 64
        assert abs(got[i] - math.cos(2 * math.pi * turns)) <= 8 * 2.0 ** -24
        assert abs(got[32 + i] - math.sin(2 * math.pi * turns)) <= 8 * 2.0 ** -24


def test_rope_in_place_and_head_major_rows(backend):
    g = torch.Generator().manual_seed(4)
    table, positions = RotaryTable(128), torch.arange(50, device="cuda") * 37
    x = torch.randn(50, 6, 128, generator=g).bfloat16().cuda()
    want = backend.rope(x, positions, table)
    fused = torch.randn(50, 8 * 128, generator=g).bfloat16().cuda()
    fused.view(50, 8, 128)[:, :6] = x
    behind = fused.view(50, 8, 128)[:, 6:].clone()
    view = fused.view(50, 8, 128)[:, :6]
    assert backend.rope(view, positions, table, out=view) is view
    assert torch.equal(view, want) and torch.equal(fused.view(50, 8, 128)[:, 6:], behind)
    head_major = torch.empty(6, 50, 128, dtype=torch.bfloat16, device="cuda").transpose(0, 1)
    backend.rope(x.transpose(0, 1).contiguous().transpose(0, 1), positions, table, out=head_major)
    assert torch.equal(head_major, want)
    odd = torch.empty(50 * 6 * 128 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(50, 6, 128)   # rows that begin off 16 bytes
    odd.copy_(x)
    assert torch.equal(backend.rope(odd, positions, table), want)


@pytest.mark.parametrize("interleaved", [False, True])
def test_gradient_is_the_transposed_map(backend, interleaved):
    # f32: <g, R(x + h e) - R(x)> = h <R^T g, e> for the linear map R, element by element of e against differences
    g = torch.Generator().manual_seed(9)
    table = RotaryTable(24, theta=100.0, magnitude=1.25)
    x, dy = torch.randn(3, 2, 32, generator=g).cuda(), torch.randn(3, 2, 32, generator=g).cuda()
    positions = torch.tensor([0, 5, 1000], device="cuda")
    dx = backend.rope(dy, positions, table, interleaved=interleaved, backward=True).cpu().double()
    base = ref.rotated(x, positions, table, interleaved)
    for d in range(32):
        step = torch.zeros_like(x, dtype=torch.float64, device="cpu")
        step[..., d] = 0.5
        change = ref.rotated(x.cpu().double() + step, positions, table, interleaved) - base
        differences = (change * dy.cpu().double()).sum(-1) / 0.5
        assert (dx[..., d] - differences).abs().max() <= 8 * 2.0 ** -24 * 1.25 * 2 * dy.abs().max().item()


def make_cache(pages, size, heads, head_dim, dtype, layout, seed):
    g = torch.Generator().manual_seed(seed)
    if layout == "rows":
        k, v = (torch.randn(pages, size, heads, head_dim, generator=g).to(dtype).cuda() for _ in range(2))
    elif layout == "heads":
        k, v = (torch.randn(pages, heads, size, head_dim, generator=g).to(dtype).cuda().transpose(1, 2) for _ in range(2))
    else:                                           # K and V of a page side by side
        both = torch.randn(pages, 2, size, heads, head_dim, generator=g).to(dtype).cuda()
        k, v = both[:, 0], both[:, 1]
    return PagedCache(k, v)


def make_batch(lengths, news, size, pages, seed, spare_rows=0, width=None):
    width = width or max(1, max(-(-n // size) for n in lengths) + 2)
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((len(lengths), width), -1, dtype=torch.int32)
    for s, n in enumerate(lengths):
        for j in range(-(-n // size)):
            table[s, j] = order.pop()
    starts = torch.tensor([0] + news, dtype=torch.int32).cumsum(0).to(torch.int32)
    batch = PagedBatch(table.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda(), starts.cuda())
    return batch, int(starts[-1]) + spare_rows


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("layout", ["rows", "heads", "pairs"])
@pytest.mark.parametrize("lengths,news,size,hq,hk,head_dim,rotary_dim", [
    ([5, 1, 0, 40], [1, 1, 0, 1], 16, 8, 2, 128, 128), ([130, 33, 64], [130, 7, 64], 32, 7, 1, 64, 48), ([9, 10], [9, 3], 3, 2, 2, 24, 8)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_append_writes_the_rows_of_its_tokens_only(backend, dtype, layout, lengths, news, size, hq, hk, head_dim, rotary_dim, interleaved):
    pages = sum(-(-n // size) for n in lengths) + 3
    cache = make_cache(pages, size, hk, head_dim, dtype, layout, 1)
    batch, tokens = make_batch(lengths, news, size, pages, 2, spare_rows=2)
    before = cache.k.clone(), cache.v.clone()
    qkv = torch.randn(tokens, (hq + 2 * hk) * head_dim, generator=torch.Generator().manual_seed(3)).to(dtype).cuda()
    table = RotaryTable(rotary_dim, theta=1000.0, scaling="linear", factor=2.0)
    out = torch.full((tokens, hq, head_dim), 7.0, dtype=dtype, device="cuda")
    backend.rope_append(qkv, cache, batch, table, q_heads=hq, interleaved=interleaved, out=out)
    backend.poll()
    rows = qkv.view(tokens, hq + 2 * hk, head_dim)
    want_k, want_v = before[0].cpu().double(), before[1].cpu()
    bound_k = torch.zeros_like(want_k)
    at = 0
    page_table = batch.page_table.cpu()
    for s, (length, n) in enumerate(zip(lengths, news)):
        for i in range(n):
            position = torch.tensor([length - n + i])
            token = rows[at:at + 1, :hq + hk]
            turned, norms = ref.rotated(token, position, table, interleaved)[0], ref.pair_norms(token, table, interleaved)[0]
            check(out[at], turned[:hq], norms[:hq], 1.0)
            page, row = int(page_table[s, int(position) // size]), int(position) % size
            want_k[page, row], bound_k[page, row] = turned[hq:], norms[hq:]
            want_v[page, row] = rows[at, hq + hk:].cpu()
            at += 1
    unit = torch.finfo(dtype).eps / 2
    assert bool(((cache.k.cpu().double() - want_k).abs() <= 8 * 2.0 ** -24 * bound_k * (1 + unit) + unit * want_k.abs() * (bound_k > 0)).all())
    assert torch.equal(cache.v.cpu(), want_v)
    assert bool((out[at:] == 7.0).all())             # tokens behind the last sequence


def test_append_with_positions_of_its_own_and_without_rotation(backend):
    cache = make_cache(8, 16, 2, 64, torch.bfloat16, "rows", 1)
    batch, tokens = make_batch([20, 30], [3, 2], 16, 8, 2)
    qkv = torch.randn(tokens, 8 * 64, device="cuda").bfloat16()
    table = RotaryTable(64)
    positions = torch.tensor([100, 7, 0, 5, 999], dtype=torch.int32, device="cuda")
    q = backend.rope_append(qkv, cache, batch, table, q_heads=4, positions=positions)
    rows = qkv.view(tokens, 8, 64)
    assert torch.equal(q, backend.rope(rows[:, :4], positions, table))
    k = backend.rope(rows[:, 4:6], positions, table)
    assert torch.equal(ref.gathered(cache.k, batch.page_table[0], 20, 16)[17:], k[:3])
    assert torch.equal(ref.gathered(cache.k, batch.page_table[1], 30, 16)[28:], k[3:])
    q = backend.rope_append(qkv, cache, batch, None, q_heads=4)
    assert torch.equal(q, rows[:, :4])
    assert torch.equal(ref.gathered(cache.k, batch.page_table[1], 30, 16)[28:], rows[3:, 4:6])


@pytest.mark.parametrize("fault", ["page too large", "page negative", "length beyond the table", "more tokens than keys"])
def test_append_leaves_out_rows_without_a_place(backend, fault):
    cache = make_cache(8, 16, 2, 64, torch.float16, "rows", 1)
    batch, tokens = make_batch([20, 30], [3, 2], 16, 8, 2)
    before = cache.k.clone(), cache.v.clone()
    good = ref.gathered(cache.k, batch.page_table[0], 20, 16).clone()
    if fault.startswith("page"):
        batch.page_table[1, 1] = 8 if fault == "page too large" else -1
    else:
        batch.key_lengths[1] = 1000 if fault.startswith("length") else 1
    qkv = torch.randn(tokens, 8 * 64, device="cuda").half()
    backend.rope_append(qkv, cache, batch, RotaryTable(64), q_heads=4)
    with pytest.raises(WB200Error, match="left out"):
        backend.poll()
    backend.poll()                                    # reported once
    now = ref.gathered(cache.k, batch.page_table[0], 20, 16)
    assert torch.equal(now[:17], good[:17]) and not torch.equal(now[17:], good[17:])
    changed = (cache.v != before[1]).flatten(1).any(1).nonzero().flatten().tolist()
    assert set(changed) <= set(batch.page_table[0, :2].tolist()) | ({int(batch.page_table[1, 0])} if fault.startswith("more") else set())


@pytest.mark.parametrize("fault", ["a range ends behind the rows", "a range begins in front of the rows", "ranges wholly behind the rows", "keys beyond the table"])
def test_append_leaves_out_whole_sequences_that_do_not_fit(backend, fault):
    """A token range or a length outside the buffers says nothing about any of its tokens: none of them is written, as attention
    reads none of them."""
    cache = make_cache(16, 16, 2, 64, torch.float16, "rows", 1)
    batch, tokens = make_batch([20, 150], [3, 2], 16, 16, 2)
    spare = (set(range(16)) - set(batch.page_table.flatten().tolist())).pop()
    batch.page_table[1, 11] = spare                   # a page for the table's last entry
    qkv = torch.randn(tokens, 8 * 64, device="cuda").half()
    if fault == "a range ends behind the rows":       # would put the rows of keys 148 and 149 at 108 and 109
        batch.query_starts[2] = tokens + 40
    elif fault == "a range begins in front of the rows":
        batch.query_starts[0] = -2
    elif fault == "ranges wholly behind the rows":
        batch.query_starts += tokens
    else:
        batch.key_lengths[1] = 12 * 16 + 1            # its first new token would still have a place
    before = cache.k.clone(), cache.v.clone()
    out = torch.full((tokens, 4, 64), 7.0, dtype=torch.float16, device="cuda")
    backend.rope_append(qkv, cache, batch, None, q_heads=4, out=out)
    with pytest.raises(WB200Error, match="left out"):
        backend.poll()
    backend.poll()
    rows, good = qkv.view(tokens, 8, 64), slice(0, 0)
    if fault in ("a range ends behind the rows", "keys beyond the table"):
        good, at = slice(0, 3), torch.arange(17, 20)
        pages = batch.page_table[0].cpu().long()[at // 16]
        before[0][pages, at % 16], before[1][pages, at % 16] = rows[:3, 4:6], rows[:3, 6:]
    elif fault == "a range begins in front of the rows":
        good, at = slice(3, 5), torch.arange(148, 150)
        pages = batch.page_table[1].cpu().long()[at // 16]
        before[0][pages, at % 16], before[1][pages, at % 16] = rows[3:, 4:6], rows[3:, 6:]
    assert torch.equal(cache.k, before[0]) and torch.equal(cache.v, before[1])
    want = torch.full_like(out, 7.0)
    want[good] = rows[good, :4]
    assert torch.equal(out, want)


@pytest.mark.parametrize("position", [1, 2, 7, 10, -1, -3])
def test_slow_pairs_keep_their_sine(backend, position):
    """(1, 0) turns into (cos t, sin t): a small sine (slow pairs, and pairs near half a turn) is right to a few units in its own
    last place: the angle is rounded once (2^-24), sincospi is off by one unit in the last place (2^-23), and the product with
    the sine is one rounding more (2^-24)."""
    slowest = RotaryTable(128, theta=500000.0, scaling="linear", factor=8.0).frequencies[-1]
    table = RotaryTable.from_frequencies([slowest, 1e-9, 3e-12, 1e-6, math.pi * (1 + 1e-7), 2 * math.pi * (1 - 1e-8), 0.3])
    n = len(table.frequencies)
    x = torch.zeros(1, 1, 2 * n, device="cuda")
    x[..., :n] = 1.0
    got = backend.rope(x, torch.tensor([position], device="cuda"), table)[0, 0].cpu().double()
    for i in range(n):
        phase = position * table._turns[i] % 2 ** 64
        half_turns, rest = divmod(phase + 2 ** 62, 2 ** 63)
        want = (-1) ** half_turns * math.sin(2 * math.pi * ((rest - 2 ** 62) / 2.0 ** 64))
        assert abs(got[n + i] - want) <= 4 * 2.0 ** -24 * abs(want), (i, got[n + i].item(), want)
