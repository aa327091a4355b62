"""What a cache held in four bits decides on the host: every refusal, without a device."""
import ctypes as C

import pytest
import torch

from tests import quantized_reference as quant
from tests.test_paged_cpu import HANDLE, INVALID, LIMIT, UNSUPPORTED, append, attention, batch
from vibe_compiler_b200 import _abi as abi
from vibe_compiler_b200.backend import B200TargetModelBackend
from vibe_compiler_b200.paged_cache import QuantizedCache


def cache(**changes):
    c = abi.QuantizedCacheDesc(pages=10, page_size=16, kv_heads=2, head_dim=64, format=abi.F16, bits=4)
    for i, rows in enumerate((c.k, c.v)):
        rows.codes, rows.steps = (1 + i) << 20, (3 + i) << 20
        rows.codes_page_stride, rows.codes_row_stride, rows.codes_head_stride = 1024, 32, 512
        rows.steps_page_stride, rows.steps_row_stride, rows.steps_head_stride = 32, 1, 16
    for name, value in changes.items():
        target, field = (getattr(c, name[0]), name[2:]) if name[:2] in ("k_", "v_") and name != "kv_heads" else (c, name)
        setattr(target, field, value)
    return c


def read(**changes):
    r = abi.CacheReadParams(k=1 << 20, v=2 << 20, k_token_stride=128, k_head_stride=64, v_token_stride=128, v_head_stride=64)
    for name, value in changes.items():
        setattr(r, name, value)
    return r


def every_call(c, b=None):
    lib, b = abi.load(), b or batch()
    one = (abi.QuantizedCacheDesc * 1)(c)
    return [lib.wb200_attention_quantized(HANDLE, C.byref(c), C.byref(b), C.byref(attention())),
            lib.wb200_rope_append_quantized(HANDLE, C.byref(c), C.byref(b), C.byref(append())),
            lib.wb200_cache_read_quantized(HANDLE, C.byref(c), C.byref(b), C.byref(read())),
            lib.wb200_pages_copy_quantized(HANDLE, one, 1, 1, 1 << 20, 1 << 20, None)]


@pytest.mark.parametrize("changes,status", [
    (dict(format=abi.F32), UNSUPPORTED), (dict(bits=8), UNSUPPORTED), (dict(bits=0), UNSUPPORTED), (dict(pages=0), INVALID), (dict(page_size=0), INVALID),
    (dict(kv_heads=0), INVALID), (dict(head_dim=0), INVALID), (dict(head_dim=60), UNSUPPORTED), (dict(head_dim=264), UNSUPPORTED),
    (dict(kv_heads=70000), LIMIT), (dict(pages=1 << 31), LIMIT),
    (dict(k_codes=None), INVALID), (dict(v_steps=None), INVALID), (dict(k_codes=(1 << 20) + 2), INVALID), (dict(v_steps=(1 << 20) + 2), INVALID),
    (dict(k_codes_row_stride=34), INVALID), (dict(v_codes_page_stride=1022), INVALID), (dict(k_codes_row_stride=28), INVALID),
    (dict(v_codes_head_stride=32), INVALID), (dict(k_steps_row_stride=0), INVALID), (dict(k_steps_page_stride=31), INVALID),
    (dict(head_dim=128), INVALID)])
def test_calls_refuse_caches(changes, status):
    assert every_call(cache(**changes)) == [status] * 4


@pytest.mark.parametrize("changes,status", [
    (dict(table_width=1 << 28), LIMIT), (dict(table_stride=4), INVALID), (dict(page_table=None), INVALID), (dict(key_lengths=None), INVALID),
    (dict(query_starts=None), INVALID), (dict(key_lengths=(2 << 20) + 2), INVALID), (dict(tokens=0), abi.OK), (dict(sequences=0), abi.OK)])
def test_calls_refuse_batches(changes, status):
    assert every_call(cache(), batch(**changes))[:3] == [status] * 3


@pytest.mark.parametrize("changes,status", [
    (dict(q_heads=0), INVALID), (dict(q_heads=3), INVALID), (dict(scale=0.0), INVALID), (dict(scale=float("nan")), INVALID), (dict(q=None), INVALID),
    (dict(out=None), INVALID), (dict(out_head_stride=32), INVALID), (dict(q=(1 << 20) + 1), INVALID), (dict(lse=(3 << 20) + 2), INVALID)])
def test_attention_refuses_arguments(changes, status):
    assert abi.load().wb200_attention_quantized(HANDLE, C.byref(cache()), C.byref(batch()), C.byref(attention(**changes))) == status


@pytest.mark.parametrize("changes,status", [
    (dict(qkv=None), INVALID), (dict(q=None), INVALID), (dict(q_token_stride=200), INVALID), (dict(positions=1 << 20, position_bytes=1), INVALID),
    (dict(q_heads=1 << 18), LIMIT), (dict(qkv=(1 << 20) + 1), INVALID)])
def test_append_refuses(changes, status):
    assert abi.load().wb200_rope_append_quantized(HANDLE, C.byref(cache()), C.byref(batch()), C.byref(append(**changes))) == status


@pytest.mark.parametrize("changes", [dict(k=None), dict(v=None), dict(k=(1 << 20) + 1), dict(k_token_stride=100), dict(v_head_stride=0)])
def test_read_refuses(changes):
    from tests.test_paged_cpu import cache as plain
    lib, b, r = abi.load(), batch(), read(**changes)
    assert lib.wb200_cache_read_quantized(HANDLE, C.byref(cache()), C.byref(b), C.byref(r)) == INVALID
    assert lib.wb200_cache_read(HANDLE, C.byref(plain()), C.byref(b), C.byref(r)) == INVALID
    assert lib.wb200_cache_read(HANDLE, C.byref(plain()), None, C.byref(r)) == INVALID
    assert lib.wb200_cache_read(HANDLE, C.byref(plain(format=abi.F32)), C.byref(b), C.byref(read())) == UNSUPPORTED


def test_copies_refuse():
    lib, word = abi.load(), 4 << 20
    two = (abi.QuantizedCacheDesc * 2)(cache(), cache(page_size=8))
    assert lib.wb200_pages_copy_quantized(HANDLE, two, 2, 1, word, word, None) == INVALID
    assert lib.wb200_pages_copy_quantized(HANDLE, two, 1, 1, None, word, None) == INVALID
    assert lib.wb200_pages_copy_quantized(HANDLE, two, 1, 1, word, word + 2, None) == INVALID
    assert lib.wb200_pages_copy_quantized(HANDLE, two, 1, 0, None, None, None) == abi.OK
    assert lib.wb200_pages_copy_quantized(None, two, 1, 0, None, None, None) == INVALID
    assert lib.wb200_attention_quantized_workspace_bytes(None, None, None, None) == 0


def test_struct_layouts_match_the_header():
    assert C.sizeof(abi.QuantizedRows) == 16 + 6 * 8
    assert C.sizeof(abi.QuantizedCacheDesc) == 24 + 2 * 64
    assert C.sizeof(abi.CacheReadParams) == 16 + 4 * 8 + 8


def test_handles_refuse():
    codes, steps = torch.zeros(4, 16, 2, 32, dtype=torch.uint8), torch.zeros(4, 16, 2, 1, 2, dtype=torch.bfloat16)
    for wrong in ((codes, steps, codes, steps), (codes.int(), steps, codes, steps), (codes, steps.float(), codes, steps.float()), (codes, steps, codes, steps.half()),
                  (codes, steps[..., 0], codes, steps), (codes, steps, codes[:, :8], steps), (codes, steps[:, :8], codes, steps)):
        with pytest.raises(ValueError):
            QuantizedCache(*wrong)
    with pytest.raises(ValueError, match="CUDA"):
        QuantizedCache(codes, steps, codes, steps)
    with pytest.raises(ValueError, match="even"):
        QuantizedCache.zeros(1, 1, 1, 7, device="cpu")


def test_calls_refuse_handles_of_another_device():
    backend = B200TargetModelBackend.__new__(B200TargetModelBackend)
    backend.device = 0

    class Elsewhere:
        device_index, shape, dtype, quantized = 1, (4, 16, 2, 64), torch.bfloat16, True
    for call in (lambda: backend.cache_read(Elsewhere, Elsewhere, 3), lambda: backend.attention_paged(torch.zeros(3, 2, 64), Elsewhere, Elsewhere, 0.1),
                 lambda: backend.rope_append(torch.zeros(3, 256), Elsewhere, Elsewhere, None, q_heads=0)):
        with pytest.raises(ValueError, match="device"):
            call()


def test_the_format_on_rows_done_by_hand():
    # range 15 in steps of one; a range that the type cannot hold a fifteenth of is rounded up
    x = torch.arange(16, dtype=torch.float32).repeat(4)[None] - 3.0
    codes, steps = quant.quantized(x.bfloat16())
    assert steps[0, 0].tolist() == [1.0, -3.0] and codes[0, :3].tolist() == [0x10, 0x32, 0x54]
    assert torch.equal(quant.values(codes, steps), x.double())
    codes, steps = quant.quantized((x / 3).bfloat16())
    step = steps[0, 0, 0].item()
    assert 1 / 3 <= step < 1 / 3 * (1 + 2.0 ** -7) and (quant.values(codes, steps) - (x / 3).bfloat16().double()).abs().max() <= step / 2


def test_each_kind_of_cache_has_its_own_scratch():
    """attention_paged takes what its own kernels need, not the larger of both kinds' scratch."""
    import types
    asked = []

    class Library:
        @staticmethod
        def wb200_attention_paged_workspace_bytes(*_):
            return 1000

        @staticmethod
        def wb200_attention_quantized_workspace_bytes(*_):
            return 3000

        @staticmethod
        def wb200_attention_paged(handle, cache, batch, p):
            asked.append(("plain", p._obj.workspace_bytes))
            return abi.OK

        @staticmethod
        def wb200_attention_quantized(handle, cache, batch, p):
            asked.append(("four bits", p._obj.workspace_bytes))
            return abi.OK
    backend = B200TargetModelBackend.__new__(B200TargetModelBackend)
    backend.device, backend._lib, backend._handle = -1, Library, None               # tensors of the CPU have no device index
    backend._empty = lambda like, shape, stream, dtype=None: torch.empty(shape, dtype=dtype or like.dtype)
    q = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    rows = types.SimpleNamespace(device_index=-1, _desc=lambda tokens: batch())
    for quantized, desc in ((True, cache()), (False, abi.PagedCacheDesc()), (True, cache()), (False, abi.PagedCacheDesc())):
        handle = types.SimpleNamespace(device_index=-1, shape=(4, 16, 2, 64), dtype=torch.bfloat16, quantized=quantized, _desc=desc)
        backend.attention_paged(q, handle, rows, 0.1, stream=0)
    assert asked == [("four bits", 3000), ("plain", 1000)] * 2
