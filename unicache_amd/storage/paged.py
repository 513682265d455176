"""The paged KV cache: 16-bit keys and values of a batch of sequences over all
layers, in pages of a common pool, the attention that reads them, and the calls that
grow, fork, cut and thin out sequences.

Beside PackedKIVICache (2/4 bits) and Block8KVCache (8 bits) this is the cache
of full precision: sequences take pages as they grow, and those that share a
prefix share its pages.  Tables, lengths, reference counts and free pages live on the device
and are changed there, so a captured graph can grow and fork sequences.  No reference counterpart:
UniCache's dense caches are contiguous tensors (storage/tensor_backend.py).
"""

from __future__ import annotations

import ctypes
import functools
import math

import torch
from torch.autograd import forward_ad

from .. import _native as nat
from ..operators.rotary import MultiAxisRotary, check_rows
from .physical import tensor_bytes

_PAGES = (16, 32, 64, 128, 256)
_ORDER = ("key", "value", "table", "lengths", "granted", "references", "free_pages")
_TENSORS = frozenset(_ORDER)
_SIZES = "Paged cache supports pages of 16, 32, 64, 128 or 256 tokens and head_dim 64 or 128"


def _check_tensor(name, t, dtype, shape, device) -> None:
    if t.dtype != dtype or tuple(t.shape) != shape or not t.is_contiguous():
        raise ValueError(f"Paged cache {name}: expected contiguous {dtype} {shape}, got {t.dtype} {tuple(t.shape)} "
                         f"strides {tuple(t.stride())}")
    if t.device != device:
        raise RuntimeError("Paged cache received tensors on different devices")


@functools.lru_cache(maxsize=256)
def _workspace_bytes(entry: str, cache: tuple, allocator: bool, query: tuple | None) -> int:
    """Workspace of an entry for the sizes of a cache and a query (the
    addresses do not matter; they are stood in for by aligned numbers)."""

    c = nat.PagedCache(*[16] * 4, *([16] * 3 if allocator else [None] * 3), *cache)
    args = [] if query is None else [nat.Block8Query(16, 0, 0, 0, *query[:2], None, *query[2:])]
    size = int(getattr(nat.lib(), entry)(c, *args))
    if size < 0:
        raise ValueError((nat.lib().uc_last_error() or b"").decode(errors="replace") or f"{entry}: bad arguments")
    return size


class PagedKVCache:
    """16-bit keys and values of S sequences over L layers, in pages of B tokens.

    The tensors, all contiguous:

    - ``key``, ``value``  [L, P, Hkv, B, D] bf16 or fp16: the pool of P pages
    - ``table``       [S, M] int32: page i of a sequence holds its tokens i * B .. i * B + B - 1; -1 for none
    - ``lengths``     [S] int32, tokens held by each sequence
    - ``granted``     [S] int32, tokens that the last reserve gave each sequence
    - ``references``  [P] int32, how many sequences hold a page
    - ``free_pages``  [ceil(P / 32)] int32, a bit for each page that none holds

    D is 64 or 128, B 16, 32, 64, 128 or 256, S 4096 at most.  Whole pages may be
    held by several sequences; a sequence's last, partly filled page (its open page) by
    no other, which the calls here see to.  Without the last three tensors the
    cache is another program's: write and attention work, the program keeps the table and lengths itself.
    Table entries that are no page hide their tokens, and nothing is written there.
    Tensors may be replaced by others of their dtype and sizes, or get other storage; calls read them where they are.

    ``max_tokens`` is how long the caller takes the longest sequence to be
    (default: the capacity; raised by reserve).  It shapes launches, and no
    result depends on its being right; only dense returns that many rows.
    The lengths are on the device, so neither replays of a captured reserve raise it
    nor do truncate, reorder and compact lower it: set it before a capture to
    what the loop will reach, and after a cut to what is left, where the caller knows.

    Tensors that track a gradient, backward or forward, are refused.  Calls
    enqueue work on the current stream of the cache's device, allocate their
    outputs and workspaces from torch's allocator and never wait for the GPU."""

    def __init__(self, key, value, table, lengths, *, granted=None, references=None, free_pages=None,
                 max_tokens=None) -> None:
        self._check(key, value, table, lengths, granted, references, free_pages)
        if max_tokens is not None and int(max_tokens) < 0:
            raise ValueError("Paged cache max_tokens must not be negative")
        self._set(key, value, table, lengths, granted, references, free_pages, max_tokens)

    @staticmethod
    def _check(key, value, table, lengths, granted, references, free_pages) -> None:
        if key.dim() != 5:
            raise ValueError("Paged cache expects keys and values [layers, pages, kv_heads, page_tokens, head_dim]")
        layers, pages, heads, b, d = map(int, key.shape)
        if key.dtype not in (torch.bfloat16, torch.float16):
            raise ValueError("Paged cache keys and values must be bf16 or fp16, both alike")
        if b not in _PAGES or d not in (64, 128):
            raise ValueError(_SIZES)
        if table.dim() != 2:
            raise ValueError("Paged cache table must be [sequences, pages]")
        s, m = map(int, table.shape)
        if not (layers and pages and heads and s and m):
            raise ValueError("Paged cache needs a layer, a page, a KV head, a sequence and a page per sequence at least")
        device = key.device
        for name, t, shape in (("key", key, tuple(key.shape)), ("value", value, tuple(key.shape))):
            _check_tensor(name, t, key.dtype, shape, device)
            check_rows(t, f"Paged cache {name}")
            if t.data_ptr() & 15:
                raise ValueError(f"Paged cache {name} must be 16-byte aligned")
        _check_tensor("table", table, torch.int32, (s, m), device)
        _check_tensor("lengths", lengths, torch.int32, (s,), device)
        kept = (granted, references, free_pages)
        if any(t is None for t in kept) != all(t is None for t in kept):
            raise ValueError("Paged cache granted, references and free_pages belong together")
        if references is not None:
            _check_tensor("granted", granted, torch.int32, (s,), device)
            _check_tensor("references", references, torch.int32, (pages,), device)
            _check_tensor("free_pages", free_pages, torch.int32, (-(-pages // 32),), device)
        if device.type != "cuda":
            raise RuntimeError(f"Paged cache requires GPU tensors (got {device})")

    def _set(self, key, value, table, lengths, granted, references, free_pages, max_tokens, grown=None) -> None:
        self.key, self.value, self.table, self.lengths = key, value, table, lengths
        self.granted, self.references, self.free_pages = granted, references, free_pages
        self.layers, self.pages, self.num_kv_heads, self.page_tokens, self.head_dim = map(int, key.shape)
        self.sequences, self.sequence_pages = map(int, table.shape)
        self.dtype, self.device = key.dtype, key.device
        self._sizes = (self.layers, self.pages, self.sequences, self.sequence_pages, self.num_kv_heads, self.head_dim,
                       self.page_tokens, nat.dtype_code(key.dtype))
        self._scale = 1.0 / math.sqrt(self.head_dim)
        self._workspaces = {}
        self.max_tokens = self.capacity if max_tokens is None else min(int(max_tokens), self.capacity)
        # tokens that were reserved in all, which a cache and its views share, and those of them that max_tokens counts
        self._grown = [0] if grown is None else grown
        self._counted = self._grown[0]
        # (refuses sizes that the kernels do not take)
        self._attention_workspace((0, self.num_kv_heads, 0, self._sizes[-1], 0))

    def __setattr__(self, name, value) -> None:
        object.__setattr__(self, name, value)
        if name in _TENSORS:  # they are checked, and their C struct is made, again
            object.__setattr__(self, "_built", None)
            object.__setattr__(self, "_reads", None)  # (which holds the tensors)

    @property
    def capacity(self) -> int:
        """Tokens that the table has room for in every sequence (the pool may have fewer)."""

        return self.sequence_pages * self.page_tokens

    @classmethod
    def empty(cls, sequences: int, pages: int, num_kv_heads: int, head_dim: int, *, layers: int = 1,
              page_tokens: int = 64, sequence_pages: int | None = None, dtype: torch.dtype = torch.bfloat16,
              device: torch.device | str = "cuda") -> "PagedKVCache":
        """A cache without tokens over a pool of `pages` free pages; a sequence
        takes `sequence_pages` of them at most (default: all)."""

        s, p, h, d, n, b = map(int, (sequences, pages, num_kv_heads, head_dim, layers, page_tokens))
        m = p if sequence_pages is None else int(sequence_pages)
        device = torch.device(device)
        if device.type != "cuda":
            raise RuntimeError(f"Paged cache requires a GPU (got {device})")
        if b not in _PAGES or d not in (64, 128):
            raise ValueError(_SIZES)
        if min(s, p, h, n, m) <= 0:
            raise ValueError("Paged cache needs a layer, a page, a KV head, a sequence and a page per sequence at least")
        if dtype not in (torch.bfloat16, torch.float16):
            raise ValueError("Paged cache keys and values must be bf16 or fp16, both alike")
        cache = cls.__new__(cls)
        key = torch.empty((n, p, h, b, d), dtype=dtype, device=device)
        counts = [torch.zeros(size, dtype=torch.int32, device=device) for size in (s, s, p)]
        words = torch.full((-(-p // 32),), -1, dtype=torch.int32, device=device)
        if p % 32:
            words[-1:].fill_((1 << p % 32) - 1)
        cache._set(key, torch.empty_like(key), torch.full((s, m), -1, dtype=torch.int32, device=device), counts[0],
                   counts[1], counts[2], words, 0)
        return cache

    def layer(self, index: int, *, sequence: int | None = None) -> "PagedKVCache":
        """One layer (of one sequence) as a cache of its own over the same tensors: to read and write, not to grow or
        fork.  A segment of run_fused_mixed_attention and run_batched_physical_attention is such a view."""

        index = self._layer(index)
        table, lengths = self.table, self.lengths
        if sequence is not None:
            sequence = int(sequence)
            if not 0 <= sequence < self.sequences:
                raise ValueError(f"Paged cache has sequences 0 .. {self.sequences - 1} (got {sequence})")
            table, lengths = table[sequence:sequence + 1], lengths[sequence:sequence + 1]
        view = type(self).__new__(type(self))
        view._set(self.key[index:index + 1], self.value[index:index + 1], table, lengths, None, None, None,
                  self.max_tokens, self._grown)
        view._counted = self._counted
        return view

    # ------------------------------------------------------------- internals --
    def _layer(self, layer) -> int:
        if layer.__class__ is not int:
            layer = int(layer)
        if not 0 <= layer < self.layers:
            raise ValueError(f"Paged cache has layers 0 .. {self.layers - 1} (got {layer})")
        return layer

    def __getstate__(self) -> dict:
        return {**self.__dict__, "_built": None, "_reads": None, "_at": None}  # (a copy's tensors lie elsewhere)

    def _struct(self, books: bool = False) -> "nat.PagedCache":
        """The C struct of the tensors where they lie now (storage can be swapped under a tensor); calls that read
        granted, references and free_pages through it ask for those with `books`."""

        if self._built is not None:
            key, value, table, lengths = self._reads[0]
            if (key(), value(), table(), lengths()) == self._at[0] and (
                    not books or tuple(read() for read in self._reads[1]) == self._at[1]):
                if self.key.requires_grad or self.value.requires_grad:  # (since then, or under no_grad till now)
                    check_rows(self.key, "Paged cache key")
                    check_rows(self.value, "Paged cache value")
                return self._built
        tensors = [getattr(self, name) for name in _ORDER]
        self._check(*tensors)
        if (*self.key.shape[:2], *self.table.shape, *self.key.shape[2:]) != (
                *self._sizes[:5], self.page_tokens, self.head_dim) or self.key.dtype != self.dtype:
            raise ValueError("Paged cache tensors may be replaced by ones of the same sizes only")
        reads = [t.data_ptr for t in tensors if t is not None]
        at = [read() for read in reads]
        self._reads, self._at = (tuple(reads[:4]), tuple(reads[4:])), (tuple(at[:4]), tuple(at[4:]))
        self._built = nat.PagedCache(*at, *[None] * (7 - len(at)), *self._sizes)
        return self._built

    def _attention_workspace(self, sizes: tuple) -> int:
        nbytes = self._workspaces.get(sizes)
        if nbytes is None:
            if len(self._workspaces) >= 256:
                self._workspaces.clear()
            nbytes = self._workspaces[sizes] = _workspace_bytes("uc_paged_attn_workspace_bytes", self._sizes, False, sizes)
        return nbytes

    def _numbers(self, t: torch.Tensor, what: str) -> torch.Tensor:
        """int32 of each sequence, on the cache's device."""

        if t.dtype != torch.int32 or not t.is_contiguous() or tuple(t.shape) != (self.sequences,):
            raise ValueError(f"Paged cache {what} must be contiguous int32 [{self.sequences}]")
        if t.device != self.device:
            raise RuntimeError(f"Paged cache {what} must be on the cache's device {self.device}")
        return t

    def _rows(self, t: torch.Tensor, what: str, heads: int | None = None):
        """Checked dense rows [S, n, H, D] as the kernels read them, and their strides."""

        shape = t.shape
        if len(shape) == 3 and self.sequences == 1:
            t = t.unsqueeze(0)
            shape = t.shape
        if (len(shape) != 4 or shape[0] != self.sequences or shape[3] != self.head_dim or not shape[2]
                or (heads is not None and shape[2] != heads)):
            raise ValueError(f"Paged cache {what}: expected [{self.sequences}, tokens, {heads or 'heads'}, "
                             f"{self.head_dim}], got {tuple(shape)}")
        if t.dtype != self.dtype:
            raise ValueError(f"Paged cache {what} must have the cache's dtype {self.dtype} (got {t.dtype})")
        if t.requires_grad or forward_ad._current_level >= 0:
            check_rows(t, f"Paged cache {what}")
        if t.device != self.device:
            raise RuntimeError(f"Paged cache {what} must be on the cache's device {self.device}")
        return nat.rows16(t)

    def _allocator(self, what: str) -> None:
        if self.references is None:
            raise RuntimeError(f"Paged cache {what} needs the pool's references and free pages")

    # ------------------------------------------------------------------ pages --
    def reserve(self, tokens: int, *, counts: torch.Tensor | None = None) -> torch.Tensor:
        """Room for `tokens` more tokens of every sequence, or the first counts[s] (int32 on
        the device) of sequence s, whose rows write then takes; all layers at once.

        Free pages go out lowest first, to the sequences in order, and `lengths` advances, on
        the device, which alone knows how far the pool goes: `granted`, which is returned, is what each
        sequence got.  `max_tokens` is raised by `tokens`; replays of a captured call do not raise it."""

        self._allocator("reserve")
        tokens = int(tokens)
        if tokens < 0 or tokens >= 1 << 30:
            raise ValueError("Paged cache reserve: tokens must not be negative, and below 2^30")
        if counts is not None:
            counts = self._numbers(counts, "counts")
        nat.call_on(self.device, "uc_paged_reserve", self._struct(True), tokens, nat.ptr(counts))
        if nat.capturing(self.device):  # (replays are not seen from here)
            self._grown[0] += 1 << 40
        self._grown[0] += tokens
        self._counted += tokens
        self.max_tokens = min(self.max_tokens + tokens, self.capacity)
        return self.granted

    def reorder(self, parents: torch.Tensor, *, lengths: torch.Tensor | None = None) -> None:
        """Sequence s becomes what sequence parents[s] (int32 on the device) was before the
        call, and empty where that is no sequence (-1): forks, the beams of a search, and freeing
        in one call.  With `lengths` it keeps its first lengths[s] tokens at most.

        Whole pages are shared.  Of the sequences with the same open page the lowest keeps it
        (unless another holds it whole), the others get copies of its rows in free pages, taken after the
        pages that nobody holds any more are freed; where none is left, a sequence ends with its whole pages."""

        self._allocator("reorder")
        parents = self._numbers(parents, "parents")
        if lengths is not None:
            lengths = self._numbers(lengths, "lengths")
        self._reorder(parents, lengths)

    def truncate(self, lengths: torch.Tensor) -> None:
        """Each sequence keeps its first lengths[s] tokens (int32 on the device) at most, as after
        drafted tokens were refused; pages behind are released.  (An open page that was shared is copied, as in reorder.)"""

        self._allocator("truncate")
        self._reorder(None, self._numbers(lengths, "lengths"))

    def _reorder(self, parents, lengths) -> None:
        nbytes = _workspace_bytes("uc_paged_reorder_workspace_bytes", self._sizes, True, None)
        ws = nat.workspace(self.device, nbytes)
        nat.call_on(self.device, "uc_paged_reorder", self._struct(True), nat.ptr(parents), nat.ptr(lengths),
                    self.max_tokens, ws.data_ptr(), nbytes)

    def compact(self, keep: torch.Tensor) -> None:
        """Each sequence keeps, in order, the tokens t with keep[s, t] (bool or uint8 [S, T], rows may
        be strided) and those from T on: the eviction of TensorCacheStorageBackend.compact over pages, for all layers.
        Tokens whose table entries are no page are dropped, whatever the mask says.

        Pages before the first that loses a token stay, shared or not.  The kept rows behind them move into free
        pages, the lowest first, to the sequences in order, and then the pages they leave are
        released.  Where the free pages do not suffice, that sequence and those after it keep all their tokens."""

        self._allocator("compact")
        if keep.dtype not in (torch.bool, torch.uint8) or keep.dim() != 2 or keep.shape[0] != self.sequences:
            raise ValueError(f"Paged cache keep must be bool or uint8 [{self.sequences}, tokens]")
        if keep.device != self.device:
            raise RuntimeError(f"Paged cache keep must be on the cache's device {self.device}")
        if keep.shape[1] and keep.stride(1) != 1:
            keep = keep.contiguous()
        nbytes = _workspace_bytes("uc_paged_compact_workspace_bytes", self._sizes, True, None)
        ws = nat.workspace(self.device, nbytes)
        nat.call_on(self.device, "uc_paged_compact", self._struct(True), keep.data_ptr(), keep.stride(0),
                    int(keep.shape[1]), self.max_tokens, ws.data_ptr(), nbytes)

    # ------------------------------------------------------------------ calls --
    def write(self, key: torch.Tensor, value: torch.Tensor, *, layer: int = 0, query: torch.Tensor | None = None,
              rotary: MultiAxisRotary | None = None, positions: torch.Tensor | None = None,
              counts: torch.Tensor | None = None) -> torch.Tensor | None:
        """Write dense rows [S, n, Hkv, D] ([n, Hkv, D] for one sequence) into a layer's
        pages, as the last granted[s] tokens of each sequence after reserve (or the last counts[s], int32
        on the device; without granted all n): row i of counts[s] is token lengths[s] - counts[s] + i.

        With `rotary` the keys are turned on the way, and so are all rows of `query` [S, n, Hq, D], which are returned;
        `positions` [axes, S, n] (int32 or int64) default to each token's place in its sequence."""

        layer = self._layer(layer)
        if key.shape != value.shape:
            raise ValueError("Paged cache write expects keys and values of one shape")
        key, k_s, k_t, k_h = self._rows(key, "keys", self.num_kv_heads)
        value, v_s, v_t, v_h = self._rows(value, "values", self.num_kv_heads)
        n = key.shape[1]
        counts = self.granted if counts is None else self._numbers(counts, "counts")
        plan = held = out = at = None
        q_s = q_t = q_h = heads = 0
        flat = False
        if rotary is not None:
            if rotary.head_dim != self.head_dim:
                raise ValueError(f"Paged cache write: the rotary is for head_dim {rotary.head_dim}")
            if rotary.device != self.device:
                raise RuntimeError(f"Paged cache write: the rotary must be on the cache's device {self.device}")
            plan, held = rotary.plan(positions, self.sequences, n)
            if query is not None:
                flat = query.dim() == 3
                query, q_s, q_t, q_h = self._rows(query, "queries")
                heads = query.shape[2]
                if query.shape[1] != n:
                    raise ValueError("Paged cache write expects as many queries as keys")
                out = nat.empty_like(query)
                at = out.data_ptr()
        elif query is not None or positions is not None:
            raise ValueError("Paged cache write takes queries and positions with a rotary")
        if n:
            nat.call_on(self.device, "uc_paged_write", self._struct(), layer, key.data_ptr(), k_s, k_t, k_h,
                        value.data_ptr(), v_s, v_t, v_h, n, nat.ptr(counts), plan, nat.ptr(query), q_s, q_t, q_h, heads,
                        at)
        return out[0] if flat else out

    def attention(self, query: torch.Tensor, *, layer: int = 0, query_lengths: torch.Tensor | None = None,
                  causal: bool = False, sm_scale: float | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """softmax(sm_scale * q K^T) V over one layer (default scale 1/sqrt(D)): query [S, Lq, Hq, D]
        ([Lq, Hq, D] for one sequence) of the cache's dtype -> out [S, Lq, Hq, D] and the natural-log
        LSE [S, Hq, Lq] in fp32.

        Sequence s has query_lengths[s] queries (int32 on the device; default
        Lq).  With causal=True they are its last tokens: row i sees the keys up
        to lengths[s] - query_lengths[s] + i.  Rows that see no key, and rows
        behind a sequence's queries, get 0 and -inf.  Keys and values that a row does not
        see never reach it, whatever they hold; an infinity among the values that it does
        see is its output in that channel (NaN for two of both signs), however small the weight.
        Rows with a logit above fp32's range, or with none but below it, are NaN.  bf16
        values above 2^90 in magnitude may overflow sums."""

        layer = self._layer(layer)
        if sm_scale is None:
            sm_scale = self._scale
        else:
            sm_scale = ctypes.c_float(float(sm_scale)).value
            if not 2.0 ** -126 <= sm_scale <= 2.0 ** 127:
                raise ValueError("Paged attention sm_scale must be 2^-126 at least, and 2^127 at most (as fp32)")
        flat = query.dim() == 3
        query, a, b, c = self._rows(query, "queries")
        shape = query.shape
        lq, hq = shape[1], shape[2]
        if hq % self.num_kv_heads:
            raise ValueError("Query heads must be divisible by the cache's KV heads")
        if query_lengths is not None:
            query_lengths = self._numbers(query_lengths, "query_lengths")
        # (in whole steps of 128 keys, so that a decode loop's sizes repeat)
        sizes = (lq, hq, (self.max_tokens + 127) & -128, self._sizes[-1], 1 if causal else 0)
        nbytes = self._attention_workspace(sizes)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=self.device) if nbytes else None
        out = nat.empty_like(query)
        lse = query.new_empty((self.sequences, hq, lq), dtype=torch.float32)
        struct = nat.Block8Query(query.data_ptr(), a, b, c, lq, hq, nat.ptr(query_lengths), *sizes[2:])
        nat.call_on(self.device, "uc_paged_attn", self._struct(), layer, struct, sm_scale, out.data_ptr(),
                    lse.data_ptr(), nat.ptr(ws), nbytes)
        return (out[0], lse[0]) if flat else (out, lse)

    def dense(self, *, layer: int = 0, tokens: int | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """Keys and values of one layer as dense [S, tokens, Hkv, D] rows, zeros behind each sequence's length.

        `tokens` defaults to max_tokens; to the capacity after a reserve was
        captured into a graph, whose replays may have passed max_tokens."""

        layer = self._layer(layer)
        if tokens is None:
            tokens = min(self.max_tokens + self._grown[0] - self._counted, self.capacity)
        else:
            tokens = int(tokens)
            if not 0 <= tokens <= self.capacity:
                raise ValueError(f"Paged cache dense: tokens must be 0 .. {self.capacity} (got {tokens})")
        shape = (self.sequences, tokens, self.num_kv_heads, self.head_dim)
        key = torch.empty(shape, dtype=self.dtype, device=self.device)
        value = torch.empty_like(key)
        if tokens:
            nat.call_on(self.device, "uc_paged_dense", self._struct(), layer, key.data_ptr(), value.data_ptr(), tokens)
        return key, value

    # ------------------------------------------------------------------ bytes --
    @property
    def resident_bytes(self) -> int:
        return sum(self.byte_breakdown.values())

    @property
    def byte_breakdown(self) -> dict[str, int]:
        return {
            "payload_bytes": tensor_bytes(self.key) + tensor_bytes(self.value),
            "scale_bytes": 0,
            "minimum_bytes": 0,
            "residual_bytes": 0,
            "indices_bytes": sum(tensor_bytes(t) for t in (self.table, self.lengths, self.granted, self.references,
                                                           self.free_pages) if t is not None),
            "score_bytes": 0,
        }
