"""What serving from a paged cache decides on the host: the rotary tables' numbers, and every refusal, without a device.

A refused call looks at no device state, so the library is given a block of zeros for its backend handle."""
import copy
import ctypes as C
import math
import pickle
from fractions import Fraction

import pytest
import torch

from vibe_compiler_b200 import _abi as abi
from vibe_compiler_b200.backend import B200TargetModelBackend
from vibe_compiler_b200.paged_cache import PagedBatch, PagedCache, RotaryTable


@pytest.mark.parametrize("table,want", [
    (RotaryTable(8, theta=10000.0), [1.0, 0.1, 0.01, 0.001]),
    (RotaryTable(8, theta=10000.0, scaling="linear", factor=4.0), [0.25, 0.025, 0.0025, 0.00025]),
    (RotaryTable(8, theta=10000.0, scaling="base", factor=8.0), [1.0, 0.1 / 2.0, 0.01 / 4.0, 0.001 / 8.0]),   # 8^(i / 3)
])
def test_frequencies(table, want):
    assert table.rotary_dim == 8 and all(abs(f - w) <= 1e-15 for f, w in zip(table.frequencies, want))


def test_wavelength_scaling_keeps_fast_pairs_and_slows_slow_ones():
    plain, scaled = RotaryTable(128, theta=500000.0), RotaryTable(128, theta=500000.0, scaling="wavelength", factor=8.0, original_length=8192)
    for f, g in zip(plain.frequencies, scaled.frequencies):
        turns = 8192 * f / (2 * math.pi)
        if turns >= 4:
            assert g == f
        elif turns <= 1:
            assert abs(g - f / 8) <= 1e-15 * f
        else:
            keep = (turns - 1) / 3
            assert abs(g - f * (keep + (1 - keep) / 8)) <= 1e-15 * f


def test_yarn_scaling_ramps_over_the_pair_index():
    plain, scaled = RotaryTable(128), RotaryTable(128, scaling="yarn", factor=16.0, original_length=4096)
    ratios = [g / f for f, g in zip(plain.frequencies, scaled.frequencies)]
    # pair i turns 4096 theta^(-i/64) / 2 pi times; 32 turns fall at pair 20.9, one at 45.03
    assert ratios[:21] == [1.0] * 21 and all(abs(r - 1 / 16) < 1e-12 for r in ratios[46:])
    assert all(abs(r - (1 - (i - 20) / 26 * 15 / 16)) < 1e-12 for i, r in enumerate(ratios) if 20 <= i <= 46)
    assert abs(scaled.magnitude - (0.1 * math.log(16.0) + 1.0)) < 1e-15


def test_turns_are_the_frequencies_in_units_of_2_to_the_minus_64():
    table = RotaryTable.from_frequencies([1.0, 0.25, 1e-7, 0.0, -0.5, 100.0])
    for f, units in zip(table.frequencies, table._turns):
        turns = Fraction(f) / Fraction(2 * math.pi)
        assert abs(Fraction(units, 2 ** 64) - turns % 1) <= abs(turns) / 2 ** 52 + Fraction(1, 2 ** 64)


@pytest.mark.parametrize("arguments", [
    dict(rotary_dim=7), dict(rotary_dim=514), dict(rotary_dim=64, theta=0.0), dict(rotary_dim=64, theta=float("inf")),
    dict(rotary_dim=64, scaling="cubic"), dict(rotary_dim=64, scaling="linear", factor=0.0),
    dict(rotary_dim=64, scaling="wavelength", factor=2.0), dict(rotary_dim=64, scaling="yarn", factor=2.0, original_length=100, low=3.0, high=2.0),
    dict(rotary_dim=2, scaling="base", factor=2.0), dict(rotary_dim=64, magnitude=float("nan"))])
def test_rotary_tables_refuse(arguments):
    with pytest.raises(ValueError):
        RotaryTable(**arguments)


def test_tensors_have_to_be_on_the_device():
    cpu = torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        PagedCache(cpu, cpu)
    with pytest.raises(ValueError):
        PagedCache(cpu, cpu[:, :8])
    with pytest.raises(ValueError):
        PagedCache(cpu.to(torch.int32), cpu.to(torch.int32))
    i32 = torch.zeros(2, 4, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        PagedBatch(i32, i32[:, 0].contiguous(), torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError, match="query_starts"):
        PagedBatch(i32, i32[:, 0].contiguous(), torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="int32"):
        PagedBatch(i32.long(), i32[:, 0].contiguous(), torch.zeros(3, dtype=torch.int32))
    backend = B200TargetModelBackend.__new__(B200TargetModelBackend)
    backend.device = 0
    x = torch.zeros(3, 2, 64)
    with pytest.raises(ValueError):
        backend.rope(x, torch.zeros(3, dtype=torch.int64), RotaryTable(64))
    with pytest.raises(ValueError):
        backend.rope(x[0], torch.zeros(3, dtype=torch.int64), RotaryTable(64))
    with pytest.raises(ValueError):
        backend.pages_free(i32, i32[:, 0].contiguous(), i32[0], torch.zeros(1, dtype=torch.int32), 16, stream=0)


def rows(**changes):
    p = abi.RopeParams()
    p.tokens, p.heads, p.head_dim, p.format, p.position_bytes = 4, 2, 64, abi.BF16, 8
    p._turns = (C.c_uint64 * 32)()
    p.table.rotary_dim, p.table.magnitude, p.table.turns = 64, 1.0, C.addressof(p._turns)
    p.positions, p.x, p.out = 1 << 20, 2 << 20, 3 << 20
    p.x_token_stride, p.x_head_stride, p.out_token_stride, p.out_head_stride = 128, 64, 128, 64
    for name, value in changes.items():
        target, field = (p.table, name[6:]) if name.startswith("table_") else (p, name)
        setattr(target, field, value)
    return p


def cache(**changes):
    c = abi.PagedCacheDesc(pages=10, page_size=16, kv_heads=2, head_dim=64, format=abi.F16, k=1 << 20, v=2 << 20, k_page_stride=2048,
                           k_row_stride=128, k_head_stride=64, v_page_stride=2048, v_row_stride=128, v_head_stride=64)
    for name, value in changes.items():
        setattr(c, name, value)
    return c


def batch(**changes):
    b = abi.PagedBatchDesc(sequences=2, table_width=5, tokens=7, max_query=0, page_table=1 << 20, key_lengths=2 << 20, query_starts=3 << 20, table_stride=5)
    for name, value in changes.items():
        setattr(b, name, value)
    return b


def attention(**changes):
    a = abi.AttentionPagedParams(q_heads=4, causal=1, scale=0.1, q=1 << 20, out=2 << 20, q_token_stride=256, q_head_stride=64, out_token_stride=256,
                                 out_head_stride=64, workspace=1 << 20, workspace_bytes=1 << 40)
    for name, value in changes.items():
        setattr(a, name, value)
    return a


def append(**changes):
    a = abi.RopeAppendParams(q_heads=4, position_bytes=4, qkv=1 << 20, q=2 << 20, qkv_token_stride=512, q_token_stride=256, q_head_stride=64)
    for name, value in changes.items():
        setattr(a, name, value)
    return a


def tables(**changes):
    t = abi.PageTablesDesc(sequences=3, table_width=4, pages=10, page_size=16, table=1 << 20, lengths=2 << 20, refs=3 << 20, table_out=1 << 20,
                           lengths_out=2 << 20, refs_out=3 << 20, table_stride=4, table_out_stride=4)
    for name, value in changes.items():
        setattr(t, name, value)
    return t


HANDLE = (C.c_uint8 * 4096)()
INVALID, UNSUPPORTED, LIMIT = abi.ERR_INVALID_ARGUMENT, abi.ERR_UNSUPPORTED, abi.ERR_LIMIT


@pytest.mark.parametrize("changes,status", [
    (dict(format=abi.I32), UNSUPPORTED), (dict(heads=0), INVALID), (dict(position_bytes=2), INVALID), (dict(table_rotary_dim=63), INVALID),
    (dict(table_rotary_dim=66), INVALID), (dict(table_turns=None), INVALID), (dict(x=None), INVALID), (dict(positions=None), INVALID),
    (dict(out_token_stride=100), INVALID), (dict(out_head_stride=0), INVALID), (dict(x=3 << 20, x_token_stride=256), INVALID),
    (dict(heads=70000), LIMIT), (dict(tokens=0), abi.OK)])
def test_rope_refuses(changes, status):
    assert abi.load().wb200_rope(HANDLE, C.byref(rows(**changes))) == status


@pytest.mark.parametrize("changes,status", [
    (dict(format=abi.F32), UNSUPPORTED), (dict(pages=0), INVALID), (dict(page_size=0), INVALID), (dict(k=None), INVALID), (dict(v_page_stride=2000), INVALID),
    (dict(k_row_stride=64), INVALID), (dict(kv_heads=3), INVALID), (dict(head_dim=60, k_head_stride=64), UNSUPPORTED),
    (dict(head_dim=264, kv_heads=1, k_row_stride=264, v_row_stride=264, k_page_stride=4224, v_page_stride=4224), UNSUPPORTED)])
def test_attention_refuses_caches(changes, status):
    assert abi.load().wb200_attention_paged(HANDLE, C.byref(cache(**changes)), C.byref(batch()), C.byref(attention())) == status


@pytest.mark.parametrize("changes,status", [
    (dict(table_width=1 << 28), LIMIT), (dict(table_stride=4), INVALID), (dict(page_table=None), INVALID), (dict(key_lengths=None), INVALID),
    (dict(query_starts=None), INVALID), (dict(tokens=0), abi.OK), (dict(sequences=0), abi.OK)])
def test_attention_refuses_batches(changes, status):
    assert abi.load().wb200_attention_paged(HANDLE, C.byref(cache()), C.byref(batch(**changes)), C.byref(attention())) == status


@pytest.mark.parametrize("changes,status", [
    (dict(q_heads=0), INVALID), (dict(q_heads=3), INVALID), (dict(scale=0.0), INVALID), (dict(scale=-1.0), INVALID), (dict(scale=float("nan")), INVALID),
    (dict(scale=float("inf")), INVALID), (dict(q=None), INVALID), (dict(out=None), INVALID), (dict(out_head_stride=32), INVALID)])
def test_attention_refuses_arguments(changes, status):
    assert abi.load().wb200_attention_paged(HANDLE, C.byref(cache()), C.byref(batch()), C.byref(attention(**changes))) == status


@pytest.mark.parametrize("changes,status", [
    (dict(qkv=None), INVALID), (dict(q=None), INVALID), (dict(q_token_stride=200), INVALID), (dict(positions=1 << 20, position_bytes=1), INVALID),
    (dict(q_heads=1 << 18), LIMIT)])
def test_append_refuses(changes, status):
    assert abi.load().wb200_rope_append(HANDLE, C.byref(cache()), C.byref(batch()), C.byref(append(**changes))) == status


@pytest.mark.parametrize("changes,status", [
    (dict(sequences=0), INVALID), (dict(sequences=16385), LIMIT), (dict(pages=0), INVALID), (dict(page_size=1 << 30), LIMIT), (dict(table=None), INVALID),
    (dict(refs_out=None), INVALID), (dict(lengths_out=None), INVALID), (dict(table_stride=3), INVALID), (dict(table_out_stride=8), INVALID)])
def test_page_calls_refuse(changes, status):
    lib, word = abi.load(), 4 << 20
    t = tables(**changes)
    assert lib.wb200_pages_reserve(HANDLE, C.byref(t), word, word) == status
    assert lib.wb200_pages_free(HANDLE, C.byref(t), 1, word) == status
    assert lib.wb200_pages_fork(HANDLE, C.byref(t), 1, word, word, word, word, word) == status
    if "lengths_out" not in changes:                 # compact leaves the lengths alone
        assert lib.wb200_pages_compact(HANDLE, C.byref(t), word, word) == status


def test_page_calls_refuse_missing_lists():
    lib, word, t = abi.load(), 4 << 20, tables()
    assert lib.wb200_pages_reserve(HANDLE, C.byref(t), None, word) == INVALID
    assert lib.wb200_pages_free(HANDLE, C.byref(t), 1, None) == INVALID
    assert lib.wb200_pages_fork(HANDLE, C.byref(t), 4, word, word, word, word, word) == INVALID       # more forks than sequences
    assert lib.wb200_pages_fork(HANDLE, C.byref(t), 1, word, None, word, word, word) == INVALID
    assert lib.wb200_pages_compact(HANDLE, C.byref(t), None, word) == INVALID
    same = (abi.PagedCacheDesc * 2)(cache(), cache(page_size=8))
    assert lib.wb200_pages_copy(HANDLE, same, 2, 1, word, word, None) == INVALID
    assert lib.wb200_pages_copy(HANDLE, same, 1, 1, None, word, None) == INVALID
    assert lib.wb200_pages_copy(HANDLE, same, 1, 0, None, None, None) == abi.OK
    for call in (lib.wb200_pages_reserve, ):
        assert call(None, C.byref(t), word, word) == INVALID
    assert lib.wb200_attention_paged(None, None, None, None) == INVALID and lib.wb200_rope(None, None) == INVALID


def test_struct_layouts_match_the_header():
    assert C.sizeof(abi.RopeTable) == 16
    assert C.sizeof(abi.RopeParams) == 16 + 16 + 3 * 8 + 4 * 8 + 8
    assert C.sizeof(abi.PagedCacheDesc) == 24 + 8 * 8
    assert C.sizeof(abi.PagedBatchDesc) == 16 + 4 * 8
    assert C.sizeof(abi.RopeAppendParams) == 8 + 16 + 3 * 8 + 4 * 8
    assert C.sizeof(abi.AttentionPagedParams) == 16 + 3 * 8 + 4 * 8 + 3 * 8
    assert C.sizeof(abi.PageTablesDesc) == 16 + 6 * 8 + 3 * 8


class RecordingBackend:
    """The backend calls of a layer's step, as shapes."""
    device = 0

    def __init__(self):
        self.rows = {}

    def rmsnorm(self, x, weight, eps):
        return x

    def gemm_epilogue(self, x, weight, epilogue=None):
        assert x.shape[0] % 8 == 0 and x.shape[1] == weight.shape[0] and x.is_contiguous()
        return x.new_zeros(x.shape[0], weight.shape[1] // (2 if epilogue is not None else 1))

    def rope_append(self, qkv, cache, batch, table, *, q_heads):
        self.rows["append"] = qkv.shape[0]
        return qkv.new_zeros(qkv.shape[0], q_heads, 16)

    def attention_paged(self, q, cache, batch, scale, out=None):
        self.rows["attention"] = q.shape[0]
        return out.copy_(q) if out is not None else q.clone()

    def residual_add(self, a, b):
        return a + b


@pytest.mark.parametrize("tokens", [1, 3, 8, 33])
def test_a_step_gives_its_tokens_and_no_more_to_the_paged_calls(tokens):
    # the rows that fill up an eight for the GEMMs are no tokens: they would choose another kernel and hide ranges that end among them
    from vibe_compiler_b200.decoder_layer import LayerConfig, ShardedDecoderLayer, random_weights
    cfg = LayerConfig(d_model=32, q_heads=2, kv_heads=1, head_dim=16, ffn=32)
    recorder = RecordingBackend()
    layer = ShardedDecoderLayer(recorder, cfg, random_weights(cfg), device=torch.device("cpu"))
    x = torch.randn(tokens, 32).bfloat16()
    assert layer.forward_paged(x, None, None, RotaryTable(16)).shape == (tokens, 32)
    assert recorder.rows == {"append": tokens, "attention": tokens}


@pytest.mark.parametrize("changes,status", [
    (dict(x=(2 << 20) + 1), INVALID), (dict(out=(3 << 20) + 1), INVALID), (dict(positions=(1 << 20) + 4), INVALID),
    (dict(positions=(1 << 20) + 2, position_bytes=4), INVALID), (dict(x=(2 << 20) + 2, format=abi.F32), INVALID)])
def test_rope_refuses_addresses_off_its_elements(changes, status):
    assert abi.load().wb200_rope(HANDLE, C.byref(rows(**changes))) == status


@pytest.mark.parametrize("target,changes", [
    (cache, dict(k=(1 << 20) + 1)), (cache, dict(v=(2 << 20) + 1)), (batch, dict(page_table=(1 << 20) + 2)), (batch, dict(key_lengths=(2 << 20) + 2)),
    (batch, dict(query_starts=(3 << 20) + 1)), (attention, dict(q=(1 << 20) + 1)), (attention, dict(out=(2 << 20) + 1)), (attention, dict(lse=(3 << 20) + 2)),
    (append, dict(qkv=(1 << 20) + 1)), (append, dict(q=(2 << 20) + 1)), (append, dict(positions=(1 << 20) + 4, position_bytes=8))])
def test_paged_calls_refuse_addresses_off_their_elements(target, changes):
    made = {f: f(**(changes if f is target else {})) for f in (cache, batch, attention, append)}
    lib = abi.load()
    if target is not append:
        assert lib.wb200_attention_paged(HANDLE, C.byref(made[cache]), C.byref(made[batch]), C.byref(made[attention])) == INVALID
    if target is not attention:
        assert lib.wb200_rope_append(HANDLE, C.byref(made[cache]), C.byref(made[batch]), C.byref(made[append])) == INVALID
    if target is cache:
        one = (abi.PagedCacheDesc * 1)(made[cache])
        assert lib.wb200_pages_copy(HANDLE, one, 1, 1, 4 << 20, 4 << 20, None) == INVALID


def test_page_calls_refuse_addresses_off_their_elements():
    lib, word, off = abi.load(), 4 << 20, (4 << 20) + 2
    for name in ("table", "lengths", "refs", "table_out", "lengths_out", "refs_out"):
        t = tables(**{name: (5 << 20) + 2})
        assert lib.wb200_pages_reserve(HANDLE, C.byref(t), word, word) == INVALID
        assert lib.wb200_pages_free(HANDLE, C.byref(t), 1, word) == INVALID
        assert lib.wb200_pages_fork(HANDLE, C.byref(t), 1, word, word, word, word, word) == INVALID
        assert lib.wb200_pages_compact(HANDLE, C.byref(t), word, word) == INVALID
    t = tables()
    for i in range(2):
        assert lib.wb200_pages_reserve(HANDLE, C.byref(t), *[off if j == i else word for j in range(2)]) == INVALID
        assert lib.wb200_pages_compact(HANDLE, C.byref(t), *[off if j == i else word for j in range(2)]) == INVALID
        one = (abi.PagedCacheDesc * 1)(cache())
        assert lib.wb200_pages_copy(HANDLE, one, 1, 1, *[off if j == i else word for j in range(2)], None) == INVALID
    assert lib.wb200_pages_free(HANDLE, C.byref(t), 1, off) == INVALID
    for i in range(5):
        assert lib.wb200_pages_fork(HANDLE, C.byref(t), 1, *[off if j == i else word for j in range(5)]) == INVALID


@pytest.mark.parametrize("again", [copy.deepcopy, lambda t: pickle.loads(pickle.dumps(t))])
def test_a_copied_rotary_table_has_constants_of_its_own(again):
    table = RotaryTable(64, theta=500000.0, scaling="yarn", factor=4.0, original_length=8192)
    other = again(table)
    assert (other.frequencies, other.magnitude, other.rotary_dim, list(other._turns)) == (table.frequencies, table.magnitude, 64, list(table._turns))
    assert other._address == C.addressof(other._turns) != table._address
