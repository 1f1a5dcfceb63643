"""Key/value cache of 8 bits and attention over it: what a decode step needs between its packed projections.

The reference has no attention (its models are the vision networks and the MLP of
Python_Jenks_Test/Jenks_Tests/QuantNetworkTest.py); the cache completes a decode step whose matrices are
``JenksQuantLinear`` layers.  Like the other operators, everything runs on the GPU through the C ABI
(``jq_kv_append``, ``jq_kv_read``, ``jq_kv_attend`` of include/jq.h, which has the formulas and the order of the codes).
"""
from __future__ import annotations

import math
import struct
from typing import Optional, Tuple

import torch

from . import _lib, ops

_FORMATS = {"int8": _lib.JQ_KV_INT8, "e4m3": _lib.JQ_KV_E4M3}
BLOCK_SIZES = (16, 32, 64, 128)
HEAD_DIMS = (64, 128)          # of attend(); append() and read() take every multiple of 32 up to 256
_TENSORS = ("keys", "values", "key_scales", "value_scales")
_pack_strides = struct.Struct("=qq").pack              # int64_t[2]
_pack_batch = struct.Struct("=QQQiiiiii").pack         # jq_kv_batch


class KVCache:
    """A pool of blocks of ``block_size`` tokens for one layer: ``keys`` and ``values`` uint8 [blocks, kv_heads, block_size,
    head_dim] (codes in the kernels' order: the last two dims only say how many there are), ``key_scales`` and
    ``value_scales`` fp32 [blocks, kv_heads].  ``KVCache.empty`` makes one; the constructor takes tensors that are there.

    Who owns which block is the caller's: every call takes ``table`` (int32 [sequences, width], the blocks of each
    sequence in order), ``lengths`` (int32 [sequences], tokens that a sequence holds, the new ones among them) and, where
    sequences have different numbers of new tokens, ``starts`` (int32 [sequences + 1]: the new tokens of sequence i are
    the rows starts[i] .. starts[i + 1] - 1; they sit at its end) with ``max_new``, which no sequence's number exceeds.
    All three stay on the device; a step can be captured in a CUDA graph and replayed with other contents.

    The tensors may be replaced (and ``fmt`` with them), moved or resized in place between calls; a copy (``copy.deepcopy``) and
    what comes back from a file have tensors of their own.  A captured step keeps the ones it was captured with."""

    def __init__(self, keys: torch.Tensor, values: torch.Tensor, key_scales: torch.Tensor, value_scales: torch.Tensor,
                 fmt: str = "int8"):
        self.keys, self.values, self.key_scales, self.value_scales, self.fmt = keys, values, key_scales, value_scales, fmt
        self._look()

    def __setattr__(self, name, value):
        object.__setattr__(self, name, value)
        if name in _TENSORS or name == "fmt":
            object.__setattr__(self, "_c", None)

    def __setstate__(self, state):
        self.__dict__.update(state)
        self._look()

    def _where(self) -> tuple:
        """Addresses and sizes of the tensors: what a change in place shows in."""
        k, v, ks, vs = self.keys, self.values, self.key_scales, self.value_scales
        return (k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), k.numel(), v.numel(), ks.numel(), vs.numel())

    def _structure(self) -> bytes:
        """jq_kv_cache of a call, of the tensors as they are now."""
        if self._c is None or self._where() != self._at:
            self._look()
        return self._c

    def _look(self) -> None:
        """Looks the tensors over; what a call needs of them."""
        self._c = None
        keys, values, key_scales, value_scales, fmt = self.keys, self.values, self.key_scales, self.value_scales, self.fmt
        if fmt not in _FORMATS:
            raise ValueError(f"unknown cache format {fmt!r}")
        if keys.dim() != 4 or keys.shape != values.shape or keys.dtype != torch.uint8 or values.dtype != torch.uint8:
            raise ValueError("keys and values are uint8 tensors of one shape [blocks, kv_heads, block_size, head_dim]")
        if key_scales.shape != keys.shape[:2] or value_scales.shape != keys.shape[:2] or \
                key_scales.dtype != torch.float32 or value_scales.dtype != torch.float32:
            raise ValueError("the scales are fp32 tensors [blocks, kv_heads]")
        tensors = (keys, values, key_scales, value_scales)
        if not all(t.is_contiguous() for t in tensors):
            raise ValueError("the cache's tensors are contiguous")
        if any(t.device != keys.device for t in tensors):
            raise ValueError("the cache's tensors are on one device")
        self.blocks, self.kv_heads, self.block_size, self.head_dim = keys.shape
        if self.blocks == 0 or self.kv_heads == 0:
            raise ValueError("a cache has at least one block and one head")
        if self.block_size not in BLOCK_SIZES:
            raise ValueError(f"block_size must be one of {BLOCK_SIZES}")
        if self.head_dim % 32 or not 32 <= self.head_dim <= 256:
            raise ValueError("head_dim must be a multiple of 32 up to 256")
        self.device = keys.device
        self._cuda = keys.is_cuda
        self._at = self._where()
        self._need = {}                # (tokens of a sequence at most, query heads) -> bytes of workspace
        self._c = bytes(_lib.jq_kv_cache(*self._at[:4], self.blocks, self.kv_heads, self.head_dim, self.block_size, _FORMATS[fmt], 0))

    @classmethod
    def empty(cls, blocks: int, kv_heads: int, head_dim: int, *, block_size: int = 64, fmt: str = "int8",
              device="cuda") -> "KVCache":
        codes = lambda: torch.full((blocks, kv_heads, block_size, head_dim), 128 if fmt == "int8" else 0,     # noqa: E731
                                   dtype=torch.uint8, device=device)
        scales = lambda: torch.ones((blocks, kv_heads), dtype=torch.float32, device=device)                   # noqa: E731
        return cls(codes(), codes(), scales(), scales(), fmt)

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.keys, self.values, self.key_scales, self.value_scales))

    def _batch(self, table, lengths, starts, tokens, max_new) -> bytes:
        """jq_kv_batch of a call, its arguments looked over."""
        n, width = table.shape if table.dim() == 2 else (-1, 0)
        if lengths.shape != (n,):
            raise RuntimeError(f"table {tuple(table.shape)} and lengths {tuple(lengths.shape)}: [sequences, width] and [sequences]")
        if table.dtype is not torch.int32 or lengths.dtype is not torch.int32 or (starts is not None and starts.dtype is not torch.int32):
            raise RuntimeError("table, lengths and starts are int32 tensors")
        if width == 0:
            raise RuntimeError("the table has no columns")
        row, column = table.stride()
        if column != 1 and width != 1 or not lengths.is_contiguous():
            raise RuntimeError("the table's rows and the lengths are contiguous")
        device = self.device
        if table.device != device or lengths.device != device:
            raise RuntimeError(f"the cache is on {device}: table, lengths and starts are too")
        if n <= 1:
            row = width
        elif row < width:
            raise RuntimeError("the table's rows lie behind one another")
        if not n and tokens:
            raise RuntimeError(f"{tokens} new tokens of no sequence")
        at = 0
        if starts is None:
            if n and tokens % n:
                raise RuntimeError(f"{tokens} new tokens of {n} sequences: starts says how many each has")
        else:
            if starts.shape != (n + 1,) or not starts.is_contiguous() or starts.device != device:
                raise RuntimeError(f"starts is a contiguous tensor [{n + 1}] on {device}")
            at = starts.data_ptr()
        if max_new is None or max_new > tokens:
            max_new = tokens
        elif max_new < 0:
            raise RuntimeError("max_new is a number of tokens")
        if max(tokens, row) > 0x7fffffff:
            raise RuntimeError(f"{tokens} new tokens, table rows {row} apart: the library counts in 32 bits")
        if not self._cuda:
            raise RuntimeError("libjq operators run on CUDA tensors only (there is no CPU path)")
        return _pack_batch(table.data_ptr(), lengths.data_ptr(), at, n, width, row, tokens, max_new, 0)

    def _rows(self, x, heads, what):
        """[..., heads, head_dim] as rows of one stride: (tensor [tokens, heads, head_dim], strides of a row and of a head)."""
        shape = x.shape
        if len(shape) < 3 or shape[-1] != self.head_dim or (shape[-2] != heads if heads else shape[-2] % self.kv_heads):
            raise RuntimeError(f"{what} is {tuple(shape)}: [tokens, {heads or 'q_heads'}, {self.head_dim}] "
                               f"with the cache's {self.kv_heads} key heads")
        if x.dtype not in ops._DT:
            raise RuntimeError(f"unsupported dtype {x.dtype}")
        if x.device != self.device:
            raise RuntimeError(f"{what} is on {x.device}, the cache on {self.device}")
        if x.is_neg():
            x = x.resolve_neg()
        if len(shape) > 3:
            x = x.reshape(-1, shape[-2], shape[-1])
        row, head, one = x.stride()
        if one != 1:
            x = x.contiguous()
            row, head, one = x.stride()
        return x, _pack_strides(row, head)

    def append(self, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor,
               starts: Optional[torch.Tensor] = None, max_new: Optional[int] = None) -> None:
        """Quantises the new tokens' ``k`` and ``v`` ([tokens, kv_heads, head_dim], or any leading dims; fp32, fp16 or bf16) into
        the places that ``table`` and ``lengths`` give them.  A block's scale grows with its largest value, and codes that
        are there already are rounded to the new one: the result depends on what is appended in one call.  Infinities
        become the largest code, NaN 0.  A block is appended to by one sequence of a call; shared blocks are full."""
        cache = self._structure()
        k, sk = self._rows(k, self.kv_heads, "k")
        v, sv = self._rows(v, self.kv_heads, "v")
        if k.shape != v.shape or k.dtype != v.dtype:
            raise RuntimeError("k and v have one shape and dtype")
        batch = self._batch(table, lengths, starts, k.shape[0], max_new)
        with ops._on(self.device):
            st = _lib.load().jq_kv_append(cache, batch, k.data_ptr(), v.data_ptr(), sk, sv, ops._DT[k.dtype],
                                          ops._stream())
        if st:
            _lib.check(st, "jq_kv_append")

    def read(self, table: torch.Tensor, lengths: torch.Tensor, last: int,
             dtype: torch.dtype = torch.float32) -> Tuple[torch.Tensor, torch.Tensor]:
        """What the codes of every sequence's last ``last`` tokens stand for: keys and values [sequences, last, kv_heads,
        head_dim], 0 before a sequence's first token."""
        if dtype not in ops._DT:
            raise RuntimeError(f"unsupported dtype {dtype}")
        if not 0 <= last <= 0x7fffffff:
            raise RuntimeError("last is a number of tokens")
        cache = self._structure()
        batch = self._batch(table, lengths, None, 0, None)
        k, v = torch.empty((2, lengths.shape[0], last, self.kv_heads, self.head_dim), dtype=dtype, device=self.device).unbind()
        with ops._on(self.device):
            st = _lib.load().jq_kv_read(cache, batch, last, k.data_ptr(), v.data_ptr(), ops._DT[dtype], ops._stream())
        if st:
            _lib.check(st, "jq_kv_read")
        return k, v

    def attend(self, q: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, starts: Optional[torch.Tensor] = None,
               max_new: Optional[int] = None, *, scale: Optional[float] = None, window: int = 0, lse: bool = False):
        """Causal attention of the new tokens' queries ``q`` ([tokens, q_heads, head_dim], or any leading dims; fp16 or bf16)
        over the cache, their own keys and values among it (append first).  ``scale`` is 1 / sqrt(head_dim) unless given;
        with a ``window`` a query sees the last ``window`` tokens up to its own.  A query that sees nothing gets zeros.
        Returns the outputs in q's shape and dtype, with ``lse`` also fp32 ln(sum(exp(scores))) [tokens, q_heads]."""
        shape, dtype = q.shape, q.dtype
        if dtype is not torch.float16 and dtype is not torch.bfloat16:
            raise RuntimeError(f"unsupported query dtype {dtype}: fp16 or bf16")
        cache = self._structure()
        if self.head_dim not in HEAD_DIMS:
            raise RuntimeError(f"attend() takes heads of {HEAD_DIMS}, the cache has {self.head_dim}")
        x, strides = self._rows(q, 0, "q")
        if scale is None:
            scale = 1.0 / math.sqrt(self.head_dim)
        elif not 1.5e-45 <= scale <= 2.3e38:             # (above 0 and, times log2(e), finite in fp32)
            raise RuntimeError("scale must be above 0 and a number of fp32")
        if window < 0:
            raise RuntimeError("window is a number of tokens, 0 for all")
        heads = shape[-2]
        tokens = x.shape[0]
        batch = self._batch(table, lengths, starts, tokens, max_new)
        lib = _lib.load()
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        sums = torch.empty(shape[:-1], dtype=torch.float32, device=self.device) if lse else None
        if starts is None:
            most = tokens // max(1, lengths.shape[0])
        else:
            most = tokens if not max_new else min(max_new, tokens)
        with ops._on(self.device):
            need = self._need.get((most, heads))
            if need is None:
                if len(self._need) >= 1024:
                    self._need.clear()
                need = lib.jq_kv_attend_workspace_bytes(cache, batch, heads)
                if need:                       # (0: refused, and so is the call below)
                    self._need[most, heads] = need
            stream = ops._stream()
            own, at, size, status = ops._parts_workspace(self.device, need, stream)
            st = lib.jq_kv_attend_status(cache, batch, x.data_ptr(), strides, heads, scale, min(window, 0x7fffffff), out.data_ptr(),
                                         ops._addr(sums), ops._DT[dtype], at, size, status, stream)
            del own
        if st:
            _lib.check(st, "jq_kv_attend_status")
        if ops._checked:
            ops.check_status()
        return (out, sums) if lse else out
