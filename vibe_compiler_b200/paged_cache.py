"""Objects of serving from a paged KV cache, as the backend's paged operators take them.

`PagedCache` is one layer's K and V cut into pages, `QuantizedCache` the same held in four bits, `PagedBatch` the new tokens of one step and where their sequences' keys
lie, `RotaryTable` the constants of a rotation. `PageTables` keeps the page table, the lengths and the page counts of a set
of sequences through the backend's book-keeping calls. Nothing is computed on the tensors here: every operator is a method
of `B200TargetModelBackend` (`rope`, `rope_append`, `cache_read`, `attention_paged`, `pages_*`) that launches library kernels.
"""
from __future__ import annotations

import ctypes as C
import math
import struct
from typing import Optional, Sequence

import torch

from . import _abi as abi

_FORMATS = {torch.bfloat16: abi.BF16, torch.float16: abi.F16, torch.float32: abi.F32}
_CACHE_PACK = struct.Struct("=6I8q").pack
_QUANTIZED_PACK = struct.Struct("=6I2Q6q2Q6q").pack
_BATCH_PACK = struct.Struct("=4I4q").pack
assert len(_QUANTIZED_PACK(*[0] * 22)) == C.sizeof(abi.QuantizedCacheDesc)
assert len(_CACHE_PACK(*[0] * 14)) == C.sizeof(abi.PagedCacheDesc) and len(_BATCH_PACK(*[0] * 8)) == C.sizeof(abi.PagedBatchDesc)


class RotaryTable:
    """Frequencies of a rotation of `rotary_dim` elements: pair i turns by theta^(-2i / rotary_dim) radians per position,
    scaled for contexts `factor` times the trained `original_length`:

      None          as it is
      "linear"      every frequency over `factor`
      "base"        theta * factor^(R / (R - 2)): the fastest pair keeps its frequency, the slowest is slowed by `factor`
      "wavelength"  pairs that turn fewer than `low` times within the original length are slowed by `factor`, those that
                    turn more than `high` times keep their frequency, in between linear in the number of turns
      "yarn"        the YaRN method: the same between the pair indices at which `high` and `low` turns fall (`low` 1, `high`
                    32 there), linear in the index, and rotated elements scaled by 0.1 ln(factor) + 1

    `magnitude` replaces the scale of the rotated elements. `RotaryTable.from_frequencies` takes radians per position."""

    def __init__(self, rotary_dim: int, theta: float = 10000.0, scaling: Optional[str] = None, factor: float = 1.0,
                 original_length: int = 0, low: float = 1.0, high: Optional[float] = None, magnitude: Optional[float] = None):
        if rotary_dim < 0 or rotary_dim % 2 or rotary_dim > 512:
            raise ValueError("rotary_dim must be even and at most 512")
        if not (theta > 0.0 and math.isfinite(theta)):
            raise ValueError("theta must be positive and finite")
        if scaling not in (None, "linear", "base", "wavelength", "yarn"):
            raise ValueError(f"unknown rotary scaling {scaling!r}")
        if scaling is not None and not (factor > 0.0 and math.isfinite(factor)):
            raise ValueError("factor must be positive and finite")
        if scaling in ("wavelength", "yarn") and original_length <= 0:
            raise ValueError(f"{scaling} scaling needs the trained original_length")
        if high is None:
            high = 32.0 if scaling == "yarn" else 4.0
        if scaling in ("wavelength", "yarn") and not 0.0 < low < high:
            raise ValueError("low must be positive and less than high")
        if scaling == "base":
            if rotary_dim <= 2:
                raise ValueError("base scaling needs more than one pair")
            theta = theta * factor ** (rotary_dim / (rotary_dim - 2))
        if scaling == "yarn" and theta <= 1.0:
            raise ValueError("yarn scaling needs theta > 1")
        frequencies = [theta ** (-2.0 * i / rotary_dim) for i in range(rotary_dim // 2)]
        if scaling == "linear":
            frequencies = [f / factor for f in frequencies]
        elif scaling == "wavelength":
            for i, f in enumerate(frequencies):
                turns = original_length * f / (2.0 * math.pi)
                keep = min(1.0, max(0.0, (turns - low) / (high - low)))
                frequencies[i] = f * (keep + (1.0 - keep) / factor)
        elif scaling == "yarn":
            def index(turns):
                return rotary_dim * math.log(original_length / (turns * 2.0 * math.pi)) / (2.0 * math.log(theta))
            first, last = max(math.floor(index(high)), 0), min(math.ceil(index(low)), rotary_dim - 1)
            for i, f in enumerate(frequencies):
                slow = min(1.0, max(0.0, (i - first) / max(last - first, 0.001)))
                frequencies[i] = f * ((1.0 - slow) + slow / factor)
            if magnitude is None:
                magnitude = 0.1 * math.log(factor) + 1.0
        self._make(frequencies, 1.0 if magnitude is None else magnitude)

    @classmethod
    def from_frequencies(cls, frequencies: Sequence[float], magnitude: float = 1.0) -> "RotaryTable":
        if len(frequencies) > 256:
            raise ValueError("at most 256 pairs")
        table = cls.__new__(cls)
        table._make([float(f) for f in frequencies], magnitude)
        return table

    def _make(self, frequencies, magnitude):
        if not all(math.isfinite(f) for f in frequencies) or not math.isfinite(magnitude):
            raise ValueError("frequencies and magnitude must be finite")
        self.frequencies, self.magnitude, self.rotary_dim = tuple(frequencies), float(magnitude), 2 * len(frequencies)
        # units of 2^-64 turns; whole turns are dropped
        self._turns = (C.c_uint64 * max(1, len(frequencies)))(*[int(round(math.ldexp(f / (2.0 * math.pi), 64))) % (1 << 64) for f in frequencies])
        self._address = C.addressof(self._turns)

    def __reduce__(self):                             # a copy's constants lie elsewhere
        return type(self).from_frequencies, (self.frequencies, self.magnitude)


class PagedCache:
    """One layer's K and V: tensors [pages, page_size, kv_heads, head_dim] on one GPU, bf16 or f16 (f32 for `pages_copy`
    only). Any strides with the head dimension innermost: a cache laid out [pages, kv_heads, page_size, head_dim] is passed
    as its transposed view."""

    __slots__ = ("_k", "_v", "_desc", "device_index", "shape", "dtype")
    quantized = False

    def __init__(self, k: torch.Tensor, v: torch.Tensor):
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype or k.dtype not in _FORMATS:
            raise ValueError("k and v must be [pages, page_size, kv_heads, head_dim] tensors of one of bfloat16 / float16 / float32")
        if not k.is_cuda or k.device != v.device:
            raise ValueError("k and v must be CUDA tensors of one device")
        if k.shape[3] > 1 and (k.stride(3) != 1 or v.stride(3) != 1):
            raise ValueError("the head dimension of k and v must be contiguous")
        self._k, self._v, self.device_index, self.shape, self.dtype = k, v, k.device.index, k.shape, k.dtype
        self._desc = abi.PagedCacheDesc.from_buffer_copy(_CACHE_PACK(
            k.shape[0], k.shape[1], k.shape[2], k.shape[3], _FORMATS[k.dtype], 0, k.data_ptr(), v.data_ptr(),
            k.stride(0), k.stride(1), k.stride(2), v.stride(0), v.stride(1), v.stride(2)))

    @classmethod
    def zeros(cls, pages: int, page_size: int, kv_heads: int, head_dim: int, dtype=torch.bfloat16, device="cuda") -> "PagedCache":
        return cls(*(torch.zeros(pages, page_size, kv_heads, head_dim, dtype=dtype, device=device) for _ in range(2)))

    # The calls pass on addresses, so a copy is made anew, and so is what they are taken from when another tensor is put in.
    def __reduce__(self):
        return type(self), (self._k, self._v)

    k = property(lambda self: self._k, lambda self, k: self.__init__(k, self._v))
    v = property(lambda self: self._v, lambda self, v: self.__init__(self._k, v))

    @property
    def page_size(self) -> int:
        return self._k.shape[1]


class QuantizedCache:
    """One layer's K and V held in four bits: codes, uint8 [pages, page_size, kv_heads, head_dim / 2], two to a byte, the even
    element in the low half, and steps [pages, page_size, kv_heads, groups, 2] of bfloat16 or float16, the pair (step, low) of
    every 64 elements (the last group of a head takes what is left): a code c stands for low + c * step. The calls that take a
    PagedCache take one of these in its place; queries and projections are of the steps' type. head_dim is a multiple of 8 up to
    256. Any strides that keep rows of codes and pairs of steps contiguous; `zeros` lays the rows of a head one behind the other
    ([pages, kv_heads, page_size, ...] in memory), which the kernels read widest."""

    __slots__ = ("_tensors", "_desc", "device_index", "shape", "dtype")
    quantized = True
    GROUP = 64

    def __init__(self, k_codes: torch.Tensor, k_steps: torch.Tensor, v_codes: torch.Tensor, v_steps: torch.Tensor):
        dtype, shape = k_steps.dtype, tuple(k_codes.shape)
        if k_codes.dtype != torch.uint8 or v_codes.dtype != torch.uint8 or len(shape) != 4 or v_codes.shape != shape:
            raise ValueError("codes must be uint8 [pages, page_size, kv_heads, head_dim / 2] tensors")
        head_dim = 2 * shape[3]
        if dtype not in (torch.bfloat16, torch.float16) or v_steps.dtype != dtype or \
                any(t.shape != (*shape[:3], -(-head_dim // self.GROUP), 2) for t in (k_steps, v_steps)):
            raise ValueError("steps must be [pages, page_size, kv_heads, groups of 64 elements, 2] tensors of bfloat16 or float16")
        device = k_codes.get_device()
        if device < 0 or any(t.get_device() != device for t in (k_steps, v_codes, v_steps)):
            raise ValueError("codes and steps must be CUDA tensors of one device")
        if any(t.stride(3) != 1 and shape[3] > 1 for t in (k_codes, v_codes)):
            raise ValueError("rows of codes must be contiguous")
        if any(t.stride(4) != 1 or (t.stride(3) != 2 and t.shape[3] > 1) or any(t.stride(i) % 2 and t.shape[i] > 1 for i in range(3)) for t in (k_steps, v_steps)):
            raise ValueError("steps must be contiguous pairs, one behind the other")
        self._tensors, self.device_index, self.shape, self.dtype = (k_codes, k_steps, v_codes, v_steps), device, (*shape[:3], head_dim), dtype
        rows = [x for codes, steps in ((k_codes, k_steps), (v_codes, v_steps))
                for x in (codes.data_ptr(), steps.data_ptr(), *codes.stride()[:3], *(n // 2 for n in steps.stride()[:3]))]
        self._desc = abi.QuantizedCacheDesc.from_buffer_copy(_QUANTIZED_PACK(*shape[:3], head_dim, _FORMATS[dtype], 4, *rows))

    @classmethod
    def zeros(cls, pages: int, page_size: int, kv_heads: int, head_dim: int, dtype=torch.bfloat16, device="cuda") -> "QuantizedCache":
        if head_dim % 2:
            raise ValueError("head_dim must be even")
        tensors = []
        for _ in range(2):
            tensors.append(torch.zeros(pages, kv_heads, page_size, head_dim // 2, dtype=torch.uint8, device=device).transpose(1, 2))
            tensors.append(torch.zeros(pages, kv_heads, page_size, -(-head_dim // cls.GROUP), 2, dtype=dtype, device=device).transpose(1, 2))
        return cls(*tensors)

    # As for PagedCache: copies and assigned tensors are what the calls read.
    def __reduce__(self):
        return type(self), self._tensors

    def _with(self, at: int, value) -> None:
        tensors = list(self._tensors)
        tensors[at] = value
        self.__init__(*tensors)

    k_codes = property(lambda self: self._tensors[0], lambda self, value: self._with(0, value))
    k_steps = property(lambda self: self._tensors[1], lambda self, value: self._with(1, value))
    v_codes = property(lambda self: self._tensors[2], lambda self, value: self._with(2, value))
    v_steps = property(lambda self: self._tensors[3], lambda self, value: self._with(3, value))

    @property
    def page_size(self) -> int:
        return self.shape[1]


class PagedBatch:
    """One step's new tokens. Sequence s brings tokens query_starts[s] .. query_starts[s + 1] - 1 and has key_lengths[s]
    keys, the new ones among them; key j lies in row j % page_size of page page_table[s, j // page_size]. All int32 CUDA
    tensors: page_table [sequences, width], key_lengths [sequences], query_starts [sequences + 1]. `max_query`: the most new
    tokens of one sequence, if known (it chooses between kernels, the results do not depend on it)."""

    __slots__ = ("_tensors", "device_index", "_fields")

    def __init__(self, page_table: torch.Tensor, key_lengths: torch.Tensor, query_starts: torch.Tensor, max_query: int = 0):
        if not page_table.dtype == key_lengths.dtype == query_starts.dtype == torch.int32:
            raise ValueError("page_table, key_lengths and query_starts must be int32")
        sequences = key_lengths.shape[0] if key_lengths.dim() == 1 else -1
        if page_table.dim() != 2 or query_starts.shape != (sequences + 1,) or page_table.shape[0] != sequences:
            raise ValueError("page_table is [sequences, width], key_lengths [sequences], query_starts [sequences + 1]")
        device = page_table.get_device()
        if device < 0 or device != key_lengths.get_device() or device != query_starts.get_device():
            raise ValueError("page_table, key_lengths and query_starts must be CUDA tensors of one device")
        width = page_table.shape[1]
        stride = page_table.stride()
        if (stride[1] != 1 and width > 1) or not key_lengths.is_contiguous() or not query_starts.is_contiguous():
            raise ValueError("rows of page_table, key_lengths and query_starts must be contiguous")
        if max_query < 0:
            raise ValueError("max_query must not be negative")
        self._tensors, self.device_index = (page_table, key_lengths, query_starts), device
        self._fields = (sequences, width, int(max_query), page_table.data_ptr(), key_lengths.data_ptr(), query_starts.data_ptr(), stride[0])

    # As for PagedCache.
    def __reduce__(self):
        return type(self), (*self._tensors, self.max_query)

    def _with(self, at: int, value) -> None:
        arguments = [*self._tensors, self.max_query]
        arguments[at] = value
        self.__init__(*arguments)

    page_table = property(lambda self: self._tensors[0], lambda self, value: self._with(0, value))
    key_lengths = property(lambda self: self._tensors[1], lambda self, value: self._with(1, value))
    query_starts = property(lambda self: self._tensors[2], lambda self, value: self._with(2, value))
    max_query = property(lambda self: self._fields[2], lambda self, value: self._with(3, value))

    def _desc(self, tokens: int) -> abi.PagedBatchDesc:
        sequences, width, max_query, table, lengths, starts, stride = self._fields
        return abi.PagedBatchDesc.from_buffer_copy(_BATCH_PACK(sequences, width, tokens, max_query, table, lengths, starts, stride))


class PageTables:
    """The page table, lengths and page counts of `sequences` sequences over a cache of `pages` pages, kept on the device and
    changed in place by the calls below (no host copy; each returns the call's device result). `caches` of the calls that
    move pages are every layer's PagedCache, or every layer's QuantizedCache."""

    def __init__(self, backend, sequences: int, width: int, pages: int, page_size: int):
        device = torch.device("cuda", backend.device)
        self.backend, self.page_size = backend, page_size
        self.table = torch.full((sequences, width), -1, dtype=torch.int32, device=device)
        self.lengths = torch.zeros(sequences, dtype=torch.int32, device=device)
        self.refs = torch.zeros(pages, dtype=torch.int32, device=device)

    @property
    def _state(self):
        return self.table, self.lengths, self.refs

    def reserve(self, wanted: torch.Tensor) -> torch.Tensor:
        """Room for wanted[s] tokens; int32[1]: 0 done, n pages too few, -1 a sequence too long."""
        return self.backend.pages_reserve(*self._state, wanted, self.page_size, out=self._state)[3]

    def fork(self, parents: torch.Tensor, children: torch.Tensor, caches) -> torch.Tensor:
        """children[i] becomes a copy of parents[i]; int32[1] as `pages_fork`."""
        _, _, _, sources, destinations, result = self.backend.pages_fork(*self._state, parents, children, self.page_size, out=self._state)
        self.backend.pages_copy(caches, sources, destinations)
        return result

    def free(self, sequences: torch.Tensor) -> None:
        self.backend.pages_free(*self._state, sequences, self.page_size, out=self._state)

    def compact(self, caches) -> None:
        """The pages in use to the front of the caches."""
        _, _, sources, destinations = self.backend.pages_compact(*self._state, self.page_size, out=(self.table, self.refs))
        self.backend.pages_copy(caches, sources, destinations)
