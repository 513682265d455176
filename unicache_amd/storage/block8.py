"""The 8-bit block-scaled KV cache: one layer's keys and values of a batch of
sequences as int8 or e4m3 codes with one fp32 scale per block of tokens and KV
head, and the attention that reads the codes.

Between PackedKIVICache's 2/4 bits and dense 16-bit rows: half of the dense
bytes, no residual window (the open block is quantized again as it fills),
lengths on the device, and prefill, decode and block-sparse attention over the
same tensors.  No reference counterpart: UniCache's 8-bit caches are
dequantized before they are attended (physical.py:452-475).

Quantization of a block: a = max(max|x|, 2^-60 L) with L = 127 (int8) or 448
(e4m3), scale = a / L, code = round(x L / a).  A block holding an infinity or a
NaN reads as NaN.  For every channel the block also keeps the largest and the
smallest key code (``key_bounds``), which bound what any query's product with
one of its keys can be: sparse_attention scores blocks by them.
"""

from __future__ import annotations

import ctypes
import functools
import math

import torch
from torch.autograd import forward_ad

from .. import _native as nat
from .physical import tensor_bytes

_CODES = {torch.int8: nat.UC_INT8, torch.float8_e4m3fn: nat.UC_E4M3}
_HALVES = (torch.bfloat16, torch.float16)


def _check_untracked(t: torch.Tensor, what: str) -> None:
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{what} requires a gradient, which the 8-bit cache does not give; detach it")
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
        raise ValueError(f"{what} carries a forward-mode gradient, which the 8-bit cache does not give; detach it")


def _check_half(t: torch.Tensor, what: str) -> None:
    if t.dtype not in _HALVES:
        raise ValueError(f"{what} must be bf16 or fp16 (got {t.dtype})")
    _check_untracked(t, what)


def _check_tensor(name, t, dtype, shape, device, align) -> None:
    if t.dtype != dtype or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"Block8 cache {name}: expected contiguous {dtype} {shape}, got {t.dtype} "
                         f"{tuple(t.shape)} strides {tuple(t.stride())}")
    if t.requires_grad or forward_ad._current_level >= 0:
        _check_untracked(t, f"Block8 cache {name}")
    if t.device != device:
        raise RuntimeError("Block8 cache received tensors on different devices")
    if t.data_ptr() & align:
        raise ValueError(f"Block8 cache {name} must be {align + 1}-byte aligned")


def _rows16(t: torch.Tensor) -> tuple[torch.Tensor, int, int, int]:
    """A [S, T, H, D] tensor as the kernels can read it -- in place where its
    channels are adjacent and its rows on 16 bytes, else a contiguous copy --
    and its first three strides."""

    if t.is_neg():
        t = t.resolve_neg()
    aligned = t.data_ptr() % 16 == 0
    if not (aligned and t.is_contiguous()):
        a, b, c, d = t.stride()
        if aligned and d == 1 and not (a % 8 or b % 8 or c % 8):
            return t, a, b, c
        t = t.contiguous()
        if t.data_ptr() % 16:
            t = t.clone(memory_format=torch.contiguous_format)
    # (a contiguous tensor's strides of dimensions of size 1 may be anything)
    _, n, h, d = t.shape
    return t, n * h * d, h * d, d


@functools.lru_cache(maxsize=256)
def _workspace_bytes(entry: str, cache: tuple, query: tuple, *args: int) -> int:
    """Workspace of an entry for the sizes of a cache and a query (the
    addresses do not matter; they are stood in for by aligned numbers)."""

    c = nat.Block8Cache(*[16] * 6, *cache)
    q = nat.Block8Query(16, 0, 0, 0, *query[:2], None, *query[2:])
    size = int(getattr(nat.lib(), entry)(c, q, *args))
    if size < 0:
        raise ValueError((nat.lib().uc_last_error() or b"").decode(errors="replace") or f"{entry}: bad arguments")
    return size


class Block8KVCache:
    """8-bit keys and values of S sequences of one layer.

    The tensors, all contiguous, N blocks of B tokens per sequence:

    - ``key_code``    [S, Hkv, N * B, D] int8 or float8_e4m3fn
    - ``value_code``  [S, Hkv, N, D, B]  the same dtype, channels outermost in a block
    - ``key_scale``, ``value_scale``  [S, Hkv, N] fp32
    - ``key_bounds``  [S, Hkv, N, 2, D] int8: the largest, then the smallest key of each
      channel, in steps of the block's largest key / 127, rounded outwards
    - ``lengths``     [S] int32, tokens held by each sequence, on the device

    D is 64 or 128, B 32, 64 or 128.  Scales are not negative (0 will do for a
    block of zeros: to attention a value scale below 2^-88, or below 2^-60 of a
    larger one that the row has seen, counts as that).  ``tail`` ([S, Hkv, 2, B, D] in the dense
    dtype, or None) holds the dense rows of each sequence's open block for
    append.  ``max_tokens`` is how long the caller takes the longest sequence
    to be (default: the capacity, raised by append); it shapes launches, and no
    result depends on its being right, so a captured graph that appends may
    outgrow it.  Only dequantize returns that many rows.

    Tensors that track a gradient, backward or forward, are refused.  Calls
    enqueue work on the current stream of the cache's device, allocate their
    outputs and workspaces from torch's allocator and never wait for the GPU."""

    def __init__(self, key_code, value_code, key_scale, value_scale, key_bounds, lengths, *, max_tokens=None,
                 tail=None) -> None:
        if key_code.dim() != 4 or value_code.dim() != 5:
            raise ValueError("Block8 cache expects key codes [S, Hkv, N * B, D] and value codes [S, Hkv, N, D, B]")
        s, h, _, d = key_code.shape
        n, b = value_code.shape[2], value_code.shape[4]
        code_dtype = key_code.dtype
        if code_dtype not in _CODES or value_code.dtype != code_dtype:
            raise ValueError("Block8 cache codes must be int8 or float8_e4m3fn, keys and values alike")
        if b not in (32, 64, 128) or d not in (64, 128):
            raise ValueError("Block8 cache supports blocks of 32, 64 or 128 tokens and head_dim 64 or 128")
        device = key_code.device
        _check_tensor("key_code", key_code, code_dtype, (s, h, n * b, d), device, 15)
        _check_tensor("value_code", value_code, code_dtype, (s, h, n, d, b), device, 15)
        _check_tensor("key_scale", key_scale, torch.float32, (s, h, n), device, 3)
        _check_tensor("value_scale", value_scale, torch.float32, (s, h, n), device, 3)
        _check_tensor("key_bounds", key_bounds, torch.int8, (s, h, n, 2, d), device, 15)
        _check_tensor("lengths", lengths, torch.int32, (s,), device, 3)
        if tail is not None:
            if tail.dtype not in _HALVES:
                raise ValueError("Block8 cache tail must be bf16 or fp16")
            _check_tensor("tail", tail, tail.dtype, (s, h, 2, b, d), device, 15)
        if device.type != "cuda":
            raise RuntimeError(f"Block8 cache requires GPU tensors (got {device})")
        if not s or not h or not n:
            raise ValueError("Block8 cache needs a sequence, a KV head and a block at least")
        if max_tokens is not None and int(max_tokens) < 0:
            raise ValueError("Block8 cache max_tokens must not be negative")
        self._set(key_code, value_code, key_scale, value_scale, key_bounds, lengths, tail, (s, h, d, n, b), max_tokens)

    def _set(self, key_code, value_code, key_scale, value_scale, key_bounds, lengths, tail, sizes, max_tokens) -> None:
        self.key_code, self.value_code = key_code, value_code
        self.key_scale, self.value_scale = key_scale, value_scale
        self.key_bounds, self.lengths, self.tail = key_bounds, lengths, tail
        self.sequences, self.num_kv_heads, self.head_dim, self.blocks, self.block_tokens = sizes
        self.code_dtype, self.device = key_code.dtype, key_code.device
        self._sizes = (*sizes, _CODES[key_code.dtype])
        self.max_tokens = self.capacity if max_tokens is None else min(int(max_tokens), self.capacity)

    @property
    def capacity(self) -> int:
        """Tokens that every sequence has room for."""

        return self.blocks * self.block_tokens

    @classmethod
    def empty(cls, sequences: int, capacity: int, num_kv_heads: int, head_dim: int, *, block_tokens: int = 64,
              code_dtype: torch.dtype = torch.float8_e4m3fn, dtype: torch.dtype = torch.bfloat16,
              device: torch.device | str = "cuda") -> "Block8KVCache":
        """A cache without tokens, with room for `capacity` of them (rounded up
        to whole blocks) in every sequence, that takes dense rows of `dtype`."""

        cache = cls._allocate(int(sequences), int(capacity), int(num_kv_heads), int(head_dim), int(block_tokens),
                              code_dtype, dtype, torch.device(device), 0)
        cache.lengths.zero_()
        return cache

    @classmethod
    def _allocate(cls, s, capacity, h, d, b, code_dtype, dtype, device, max_tokens) -> "Block8KVCache":
        if device.type != "cuda":
            raise RuntimeError(f"Block8 cache requires a GPU (got {device})")
        if capacity <= 0 or s <= 0 or h <= 0:
            raise ValueError("Block8 cache needs a sequence, a KV head and a token of capacity at least")
        if b not in (32, 64, 128) or d not in (64, 128):
            raise ValueError("Block8 cache supports blocks of 32, 64 or 128 tokens and head_dim 64 or 128")
        if code_dtype not in _CODES:
            raise ValueError("Block8 cache codes must be int8 or float8_e4m3fn")
        if dtype not in _HALVES:
            raise ValueError("Block8 cache tail must be bf16 or fp16")
        n = -(-capacity // b)
        cache = cls.__new__(cls)
        cache._set(
            torch.empty((s, h, n * b, d), dtype=code_dtype, device=device),
            torch.empty((s, h, n, d, b), dtype=code_dtype, device=device),
            torch.empty((s, h, n), dtype=torch.float32, device=device),
            torch.empty((s, h, n), dtype=torch.float32, device=device),
            torch.empty((s, h, n, 2, d), dtype=torch.int8, device=device),
            torch.empty((s,), dtype=torch.int32, device=device),
            torch.empty((s, h, 2, b, d), dtype=dtype, device=device), (s, h, d, n, b), max_tokens)
        return cache

    @classmethod
    def from_dense(cls, key: torch.Tensor, value: torch.Tensor, *, lengths: torch.Tensor | None = None,
                   capacity: int | None = None, block_tokens: int = 64,
                   code_dtype: torch.dtype = torch.float8_e4m3fn) -> "Block8KVCache":
        """Quantize dense [S, T, Hkv, D] (or [T, Hkv, D], one sequence) keys and
        values; sequence s holds its first lengths[s] rows (int32 on the device, copied;
        default: all).  `capacity` (default T) is the tokens each sequence has room for."""

        if key.dim() == 3:
            key, value = key.unsqueeze(0), value.unsqueeze(0)
        if key.shape != value.shape or key.dim() != 4:
            raise ValueError("Block8 cache expects matching [sequences, tokens, kv_heads, head_dim] tensors")
        if key.dtype != value.dtype:
            raise ValueError("Block8 cache expects key and value of one dtype")
        _check_half(key, "Block8 keys")
        _check_half(value, "Block8 values")
        device = nat.require_device(key, value, lengths, what="Block8 cache")
        s, t, h, d = key.shape
        capacity = max(t, 1) if capacity is None else int(capacity)
        if capacity < t:
            raise ValueError("Block8 cache capacity must cover the tokens")
        if lengths is not None and (lengths.dtype != torch.int32 or tuple(lengths.shape) != (s,)
                                    or not lengths.is_contiguous()):
            raise ValueError("Block8 cache lengths must be contiguous int32 [sequences]")
        cache = cls._allocate(s, capacity, h, d, int(block_tokens), code_dtype, key.dtype, device, t)
        if t:
            (key, *k_strides), (value, *v_strides) = _rows16(key), _rows16(value)
            cache._call("uc_block8_pack", cache._struct(), key.data_ptr(), *k_strides, value.data_ptr(), *v_strides,
                        nat.dtype_code(key.dtype), t, nat.ptr(lengths), cache.tail.data_ptr())
        else:
            cache.lengths.zero_()
        return cache

    # ------------------------------------------------------------- internals --
    def _struct(self) -> "nat.Block8Cache":
        return nat.Block8Cache(self.key_code.data_ptr(), self.value_code.data_ptr(), self.key_scale.data_ptr(),
                               self.value_scale.data_ptr(), self.key_bounds.data_ptr(), self.lengths.data_ptr(),
                               *self._sizes)

    def _call(self, entry: str, *args) -> None:
        """An entry point on the current stream of the cache's device, whatever
        the current device is."""

        stream = nat.stream(self.device)
        if self.device.index == torch.cuda.current_device():
            nat.call(entry, *args, stream)
        else:
            with torch.cuda.device(self.device):
                nat.call(entry, *args, stream)

    def _query(self, query, query_lengths, causal):
        """The checked query as the kernels read it, its struct, and its sizes."""

        if query.dim() == 3 and self.sequences == 1:
            query = query.unsqueeze(0)
        if query.dim() != 4 or query.shape[0] != self.sequences or query.shape[3] != self.head_dim:
            raise ValueError(f"Block8 attention expects queries [{self.sequences}, tokens, heads, {self.head_dim}], "
                             f"got {tuple(query.shape)}")
        _, lq, hq, _ = query.shape
        if hq == 0 or hq % self.num_kv_heads:
            raise ValueError("Query heads must be divisible by the cache's KV heads")
        _check_half(query, "Block8 queries")
        if query_lengths is not None and (query_lengths.dtype != torch.int32 or not query_lengths.is_contiguous()
                                          or tuple(query_lengths.shape) != (self.sequences,)):
            raise ValueError("Block8 query_lengths must be contiguous int32 [sequences]")
        if query.device != self.device or (query_lengths is not None and query_lengths.device != self.device):
            raise RuntimeError(f"Block8 attention requires GPU tensors on the cache's device {self.device}")
        query, a, b, c = _rows16(query)
        dtype, causal = nat.dtype_code(query.dtype), 1 if causal else 0
        struct = nat.Block8Query(query.data_ptr(), a, b, c, lq, hq, nat.ptr(query_lengths), self.max_tokens, dtype, causal)
        return query, struct, (lq, hq, self.max_tokens, dtype, causal)

    def _scale(self, sm_scale) -> float:
        sm_scale = 1.0 / math.sqrt(self.head_dim) if sm_scale is None else ctypes.c_float(float(sm_scale)).value
        if not 0.0 < sm_scale <= 2.0 ** 127:
            raise ValueError("Block8 attention sm_scale must be positive, and 2^127 at most (as fp32)")
        return sm_scale

    def _attend(self, cache, query, struct, sizes, blocks, budget, query_block, sm_scale, ws, nbytes):
        lq, hq = sizes[0], sizes[1]
        out = torch.empty_like(query, memory_format=torch.contiguous_format)
        lse = torch.empty((self.sequences, hq, lq), dtype=torch.float32, device=self.device)
        self._call("uc_block8_attn", cache, struct, nat.ptr(blocks), budget, query_block, sm_scale, out.data_ptr(),
                   lse.data_ptr(), nat.ptr(ws), nbytes)
        return out, lse

    # ------------------------------------------------------------------ calls --
    def append(self, key: torch.Tensor, value: torch.Tensor, *, counts: torch.Tensor | None = None) -> None:
        """Append dense rows [S, n, Hkv, D] ([n, Hkv, D] for one sequence) to
        the sequences: the first counts[s] of them (int32 on the device; default all n).  The
        result equals from_dense of all rows.  `lengths` advances on the device,
        which alone knows them: rows past the capacity are dropped there."""

        if self.tail is None:
            raise RuntimeError("Block8 append needs the open blocks' dense rows (tail)")
        if key.dim() == 3 and self.sequences == 1:
            key, value = key.unsqueeze(0), value.unsqueeze(0)
        if (key.shape != value.shape or key.dim() != 4
                or (int(key.shape[0]), *map(int, key.shape[2:])) != (self.sequences, self.num_kv_heads, self.head_dim)):
            raise ValueError("Block8 append expects [sequences, tokens, kv_heads, head_dim] K/V matching the cache")
        if key.dtype != self.tail.dtype or value.dtype != self.tail.dtype:
            raise ValueError(f"Block8 append expects K/V in the tail's dtype {self.tail.dtype}")
        _check_half(key, "Block8 keys")
        _check_half(value, "Block8 values")
        if counts is not None and (counts.dtype != torch.int32 or not counts.is_contiguous()
                                   or tuple(counts.shape) != (self.sequences,)):
            raise ValueError("Block8 append counts must be contiguous int32 [sequences]")
        if nat.require_device(key, value, counts, what="Block8 append") != self.device:
            raise RuntimeError("Block8 append received tensors on different devices")
        n = int(key.shape[1])
        if n == 0:
            return
        (key, *k_strides), (value, *v_strides) = _rows16(key), _rows16(value)
        self._call("uc_block8_append", self._struct(), self.tail.data_ptr(), key.data_ptr(), *k_strides,
                   value.data_ptr(), *v_strides, nat.dtype_code(key.dtype), n, nat.ptr(counts))
        self.max_tokens = min(self.max_tokens + n, self.capacity)

    def dequantize(self, dtype: torch.dtype | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """Keys and values as dense [S, max_tokens, Hkv, D] rows of `dtype`
        (default: the tail's, bf16 without one), zeros behind each sequence's length."""

        dtype = dtype or (self.tail.dtype if self.tail is not None else torch.bfloat16)
        if dtype not in _HALVES:
            raise ValueError(f"Block8 dequantization restores bf16 or fp16 (got {dtype})")
        shape = (self.sequences, self.max_tokens, self.num_kv_heads, self.head_dim)
        key = torch.empty(shape, dtype=dtype, device=self.device)
        value = torch.empty_like(key)
        if self.max_tokens:
            self._call("uc_block8_dequant", self._struct(), key.data_ptr(), value.data_ptr(), nat.dtype_code(dtype),
                     self.max_tokens)
        return key, value

    def attention(self, query: torch.Tensor, *, query_lengths: torch.Tensor | None = None, causal: bool = False,
                  sm_scale: float | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """softmax(sm_scale * q K^T) V over the whole cache (default scale
        1/sqrt(D)): query [S, Lq, Hq, D] ([Lq, Hq, D] for one sequence) of bf16 or
        fp16 -> out [S, Lq, Hq, D] and the natural-log LSE [S, Hq, Lq] in fp32.

        Sequence s has query_lengths[s] queries (int32 on the device; default
        Lq).  With causal=True they are its last tokens: row i sees the keys up
        to lengths[s] - query_lengths[s] + i.  Rows that see no key, and rows
        behind a sequence's queries, get 0 and -inf."""

        sm_scale = self._scale(sm_scale)
        q, struct, sizes = self._query(query, query_lengths, causal)
        nbytes = _workspace_bytes("uc_block8_attn_workspace_bytes", self._sizes, sizes, 0, 0)
        ws = nat.workspace(self.device, nbytes) if nbytes else None
        return self._attend(self._struct(), q, struct, sizes, None, 0, 0, sm_scale, ws, nbytes)

    def sparse_attention(self, query: torch.Tensor, *, budget: int, query_block: int = 1, sink: int = 1,
                         recent: int = 1, query_lengths: torch.Tensor | None = None, causal: bool = False,
                         sm_scale: float | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """attention() over `budget` blocks of each KV head, chosen for each run
        of `query_block` query tokens: the first `sink` blocks, the blocks from
        the one `recent` - 1 before the run's own first block on, and of the
        others those in which a key inside the bounds can have the largest
        product with one of the run's rows (queries rounded to 8 bits; the lower
        index of equals).  A run takes the time of `budget` blocks, whether its
        sequence has as many or not.  Returns out, lse and the chosen blocks, int32
        [S, ceil(Lq / query_block), Hkv, budget], ascending, then -1."""

        budget, query_block, sink, recent = int(budget), int(query_block), int(sink), int(recent)
        if budget <= 0 or query_block <= 0:
            raise ValueError("Block8 sparse attention needs a positive budget and query_block")
        if budget > (1 << 30) // self.block_tokens:
            raise ValueError("Block8 sparse attention: a budget of more than 2^30 tokens")
        if not 0 <= sink <= budget or not 1 <= recent <= budget:
            raise ValueError("Block8 sparse attention: sink must not be negative, recent must be positive, and neither "
                             "more than the budget")
        sm_scale = self._scale(sm_scale)
        q, struct, sizes = self._query(query, query_lengths, causal)
        query_block = min(query_block, max(sizes[0], 1))
        # one workspace, for the one call and then for the other
        nbytes = max(_workspace_bytes("uc_block8_select_workspace_bytes", self._sizes, sizes, query_block),
                     _workspace_bytes("uc_block8_attn_workspace_bytes", self._sizes, sizes, budget, query_block))
        runs = -(-sizes[0] // query_block)
        blocks = torch.empty((self.sequences, runs, self.num_kv_heads, budget), dtype=torch.int32, device=self.device)
        ws = nat.workspace(self.device, nbytes)
        cache = self._struct()
        self._call("uc_block8_select", cache, struct, budget, sink, recent, query_block, blocks.data_ptr(),
                   ws.data_ptr(), nbytes)
        out, lse = self._attend(cache, q, struct, sizes, blocks, budget, query_block, sm_scale, ws, nbytes)
        return out, lse, blocks

    # ------------------------------------------------------------------ bytes --
    @property
    def resident_bytes(self) -> int:
        return sum(tensor_bytes(t) for t in (self.key_code, self.value_code, self.key_scale, self.value_scale,
                                             self.key_bounds, self.lengths, self.tail))

    @property
    def byte_breakdown(self) -> dict[str, int]:
        return {
            "payload_bytes": tensor_bytes(self.key_code) + tensor_bytes(self.value_code),
            "scale_bytes": tensor_bytes(self.key_scale) + tensor_bytes(self.value_scale),
            "minimum_bytes": 0,
            "residual_bytes": tensor_bytes(self.tail),
            "indices_bytes": tensor_bytes(self.lengths),
            "score_bytes": tensor_bytes(self.key_bounds),
        }

    @property
    def full_precision_bytes(self) -> int:
        """Bytes of the capacity's tokens as 16-bit keys and values."""

        return self.sequences * self.capacity * self.num_kv_heads * self.head_dim * 2 * 2
