"""Serving operators of the dense attention layers: a prompt's attention, and a paged
K/V cache held in 8 bits with the attention of single tokens over it.

* ``prompt_attention``: causal attention over packed prompts of different lengths,
  grouped heads, one launch;
* ``PagedKVCache``: pages of 64 tokens from one stack shared by all requests and layers,
  taken and returned in a deterministic order as the SDM pools take rows.  ``resize`` moves
  every request to a target length and gives the block tables and slot maps of the new
  tokens, ``store`` quantises their keys and values, ``attend`` answers one query token
  per request, ``read`` gives stored values back.

The reference keeps a fixed-capacity cache in the activation type for these layers
(copy_on_write_sdm/inference.py:293-306, model.py:127-185) and has no counterpart.
Serving only: no operator here has a backward pass, and inputs that ask for one are refused.
Every operation runs through ``libcowsdm.so`` (sm_100a) on the current stream; it
neither synchronises nor allocates anything but its results and, once, its workspace.
"""

from __future__ import annotations

import ctypes
import operator
from dataclasses import dataclass, field, replace
from typing import Sequence

import torch
from torch.autograd import forward_ad

from . import _lib

PAGE_TOKENS = 64
MAX_REQUESTS = 8192
HEAD_WIDTHS = (32, 64, 96, 128)
MAX_GROUP = 64  # query heads to a key head, prompt attention

_STATUS_TEXT = [
    (_lib.ST_SLAB_EXHAUSTED, "the K/V cache has no free page left"),
    (_lib.ST_INDEX_RANGE, "a request's length lies outside its block table"),
    (_lib.ST_PLAN_TOKENS, "a resize adds more tokens than were announced"),
    (_lib.ST_ROW_RANGE, "a block table holds no page for a cached token"),
    (_lib.ST_WAIT_TIMEOUT, "a bounded wait in an attention kernel gave up: the rows it was for are NaN"),
]


_ENTRIES: dict[str, object] = {}
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _call(device: torch.device, what: str, *args) -> None:
    """One entry point on the device's current stream, the device made current where it is not."""
    fn = _ENTRIES.get(what)
    if fn is None:
        fn = _ENTRIES[what] = getattr(_lib.load(), what)
    if device.index == _current_device():
        rc = fn(*args, _lib.stream_of(device))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, _lib.stream_of(device))
    if rc:
        _lib.check(rc, what)


def _rows(t: torch.Tensor, what: str) -> tuple[torch.Tensor, int, int]:
    """``t`` [n, heads, width] with rows the kernels can read, contiguous and on 16-byte boundaries (a
    copy where it is not so), and its strides; those of a dimension of one are made up."""
    if not t.is_cuda:
        _lib.require_cuda(t, what)
    if (t.requires_grad and torch.is_grad_enabled()) or (forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None):
        raise ValueError(f"{what} asks for a gradient: the serving attention has no backward pass")
    n, heads, width = t.shape
    s0, s1, s2 = t.stride()
    if heads == 1:
        s1 = width
    if n == 1:
        s0 = heads * width
    mask = 3 if t.element_size() == 4 else 7
    if s2 == 1 and s0 > 0 and s1 > 0 and not (s0 | s1) & mask and not t.data_ptr() & 15:
        return t, s0, s1
    return t.clone(memory_format=torch.contiguous_format), heads * width, width


def _not_capturing(what: str) -> None:
    """Raise where a buffer that is kept would be made inside a graph capture: its zeroing would be a node of the graph, and
    calls before the first replay would find it as the allocator left it."""
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"{what} must be made before the capture: call it once outside")


_PROMPT_STATUS: dict[int, torch.Tensor] = {}


def prompt_attention_status(device: torch.device) -> torch.Tensor:
    """The device's status word of ``prompt_attention`` calls without one of their own: 0, or ``_lib.ST_WAIT_TIMEOUT`` once a
    wait inside the kernel gave up and made rows NaN.  Who reads it may zero it.  It is made at the device's first call,
    which must not be inside a graph capture."""
    word = _PROMPT_STATUS.get(device.index)
    if word is None:
        _not_capturing("the status word of prompt attention (prompt_attention_status)")
        word = _PROMPT_STATUS[device.index] = torch.zeros((), dtype=torch.int32, device=device)
    return word


def prompt_attention(queries: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, starts: torch.Tensor, *,
                     scale: float | None = None, status: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention over packed prompts.

    ``queries`` ``[tokens, heads, width]``, ``keys`` and ``values`` ``[tokens, kv_heads,
    width]`` (float32, bfloat16 or float16, any strides with contiguous rows); sequence b
    holds tokens ``starts[b] .. starts[b+1]-1`` (int32, ascending, on the device).  Token i
    attends to its own sequence's tokens up to itself with ``softmax(scale * q . k)``, ``scale``
    1 / sqrt(width) by default; ``heads / kv_heads`` neighbouring query heads share a key head.
    Returns ``[tokens, heads, width]``; rows of tokens outside every sequence are unspecified.

    Sums and softmax statistics are float32; 16-bit inputs have their weights rounded to their type before
    they meet the values.  ``status`` (an int32 device word, a cache's ``status_word`` for one; ``prompt_attention_status``
    by default) collects a wait that gave up, whose rows are NaN.
    """
    if queries.ndim != 3 or keys.ndim != 3 or keys.shape != values.shape:
        raise ValueError("prompt attention takes queries, keys and values [tokens, heads, width]")
    tokens, heads, width = queries.shape
    kv_heads = keys.shape[1]
    if keys.shape[0] != tokens or keys.shape[2] != width or kv_heads < 1 or heads % kv_heads:
        raise ValueError("queries, keys and values do not match")
    if heads < 1 or width < 1 or width % 8 or width > 128 or heads // kv_heads > MAX_GROUP:
        raise ValueError(f"prompt attention takes widths of 8, 16 .. 128 and up to {MAX_GROUP} query heads to a key head")
    if not queries.dtype == keys.dtype == values.dtype:
        raise ValueError("queries, keys and values must share one dtype")
    code = _lib.dtype_code(queries.dtype)
    (q, q0, q1), (k, k0, k1), (v, v0, v1) = _rows(queries, "queries"), _rows(keys, "keys"), _rows(values, "values")
    device = q.device
    if k.device != device or v.device != device or starts.device != device:
        raise ValueError("queries, keys, values and starts must be on one device")
    if starts.dtype != torch.int32 or starts.ndim != 1 or starts.numel() < 1 or not starts.is_contiguous():
        raise ValueError("starts must be a contiguous int32 vector [sequences + 1]")
    if status is None:
        status = prompt_attention_status(device)
    elif status.dtype != torch.int32 or status.numel() != 1 or status.device != device:
        raise ValueError("status must be one int32 on the inputs' device")
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    _call(device, "cow_prompt_attention", q.data_ptr(), q0, q1, k.data_ptr(), k0, k1, v.data_ptr(), v0, v1, starts.data_ptr(), starts.numel() - 1, tokens, heads, kv_heads, width,
          code, width ** -0.5 if scale is None else float(scale), out.data_ptr(), status.data_ptr())
    return out


class PagePlan:
    """Where a resize put the new tokens: ``starts`` ``[requests + 1]`` (their packed
    order, request by request), ``slots`` and ``positions`` ``[tokens]`` (``64 * page +
    offset`` in the cache, place in the request; -1 past the new tokens), all int32 on
    the device, and ``pieces`` (the new tokens page by page) for ``store``."""

    __slots__ = ("cache", "epoch", "requests", "tokens", "buffer", "_views")

    def __init__(self, cache: "PagedKVCache", epoch: int, tokens: int, buffer: torch.Tensor) -> None:
        self.cache, self.epoch, self.tokens, self.buffer = cache, epoch, tokens, buffer
        self.requests = cache.requests
        self._views = None

    def _parts(self) -> tuple[torch.Tensor, ...]:
        if self._views is None:
            tail = (self.requests + 1, self.tokens, self.tokens)
            self._views = self.buffer.split_with_sizes((4, self.buffer.numel() - 4 - sum(tail), *tail))
        return self._views

    @property
    def starts(self) -> torch.Tensor:
        return self._parts()[2]

    @property
    def slots(self) -> torch.Tensor:
        return self._parts()[3]

    @property
    def positions(self) -> torch.Tensor:
        return self._parts()[4]

    @property
    def pieces(self) -> torch.Tensor:
        """``[max pieces, 4]``: first packed token, tokens, page, offset; the first ``buffer[0]`` are set."""
        return self._parts()[1].view(-1, 4)


@dataclass(frozen=True, eq=False)
class PagedKVCache:
    """K/V of a batch of requests for ``layers`` attention layers, in pages of 64 tokens.

    Keys and values are e4m3 codes with one power-of-two scale per (layer, page, head): a
    value is ``code * scale``.  ``value_pages`` hold a page's tokens side by side, and ``key_pages`` of
    width 128 the rows of odd tokens with their halves exchanged (``read`` undoes both).  A page
    id stands for one page in every layer, so one ``resize`` serves them all.
    ``free_pages`` is a stack with its top at ``free_count - 1``.  ``status_word`` collects
    device errors as the SDM pools' ``overflow_flag`` does; ``validate_invariants`` raises.
    """

    key_pages: torch.Tensor      # [layers, pages, kv_heads, 64, head_width] float8_e4m3fn
    value_pages: torch.Tensor    # [layers, pages, kv_heads, head_width, 64] float8_e4m3fn
    key_scales: torch.Tensor     # [layers, pages, kv_heads] float32
    value_scales: torch.Tensor   # [layers, pages, kv_heads] float32
    block_tables: torch.Tensor   # [requests, max_blocks] int32
    lengths: torch.Tensor        # [requests] int32
    free_pages: torch.Tensor     # [pages] int32
    free_count: torch.Tensor     # int32
    status_word: torch.Tensor    # int32
    ticket: torch.Tensor         # int32
    _epoch: list = field(default_factory=lambda: [0], repr=False)

    @classmethod
    def allocate(cls, *, requests: int, pages: int, kv_heads: int, head_width: int, max_blocks: int, layers: int = 1,
                 device: torch.device | str = "cuda") -> "PagedKVCache":
        """An empty cache: ``requests`` block tables of ``max_blocks`` pages of 64 tokens, over ``pages`` pages."""
        if requests < 0 or pages < 0 or kv_heads < 1 or max_blocks < 0 or layers < 1:
            raise ValueError("K/V cache sizes are invalid")
        if head_width not in HEAD_WIDTHS:
            raise ValueError(f"the 8-bit K/V cache takes head widths {HEAD_WIDTHS}")
        if requests > MAX_REQUESTS or requests * max_blocks >= 1 << 25 or pages >= 1 << 25 or kv_heads > 1024:
            raise ValueError("the K/V cache exceeds the compiled limits (8192 requests, 2^25 pages and table entries)")
        device = torch.device(device)
        if device.type != "cuda":
            raise ValueError("the paged K/V cache must be on a CUDA device: it runs only through the sm_100a kernels")
        if device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())

        def zeros(*shape, dtype=torch.int32):
            return torch.zeros(shape, dtype=dtype, device=device)

        codes = (layers, pages, kv_heads, PAGE_TOKENS, head_width)
        return cls(
            key_pages=zeros(*codes, dtype=torch.uint8).view(torch.float8_e4m3fn),
            value_pages=zeros(layers, pages, kv_heads, head_width, PAGE_TOKENS, dtype=torch.uint8).view(torch.float8_e4m3fn),
            key_scales=zeros(layers, pages, kv_heads, dtype=torch.float32),
            value_scales=zeros(layers, pages, kv_heads, dtype=torch.float32),
            block_tables=torch.full((requests, max_blocks), -1, dtype=torch.int32, device=device),
            lengths=zeros(requests), free_pages=torch.arange(pages, dtype=torch.int32, device=device),
            free_count=torch.tensor(pages, dtype=torch.int32, device=device), status_word=zeros(), ticket=zeros())

    def __post_init__(self) -> None:
        # The tensors are fixed for this object's life: sizes and the C descriptor are taken once.
        layers, pages, kv_heads, _, width = self.key_pages.shape
        requests, max_blocks = self.block_tables.shape
        desc = _lib.CowKVPages(
            *(t.data_ptr() for t in (self.key_pages, self.value_pages, self.key_scales, self.value_scales, self.block_tables,
                                     self.lengths, self.free_pages, self.free_count, self.status_word, self.ticket)),
            requests, max_blocks, pages, layers, kv_heads, width)
        for name, value in (("device", self.lengths.device), ("requests", requests), ("layers", layers), ("pages", pages),
                            ("kv_heads", kv_heads), ("head_width", width), ("max_blocks", max_blocks), ("_desc", desc),
                            ("_at", ctypes.addressof(desc)), ("_workspaces", {})):
            object.__setattr__(self, name, value)

    def storage_bytes(self) -> dict[str, int]:
        """Bytes reserved for codes and scales, and for tables and stack."""
        pools = (self.key_pages, self.value_pages, self.key_scales, self.value_scales)
        meta = (self.block_tables, self.lengths, self.free_pages, self.free_count, self.status_word, self.ticket)
        return {"kv_pages": sum(t.numel() * t.element_size() for t in pools),
                "kv_metadata": sum(t.numel() * t.element_size() for t in meta)}

    # ---- operators

    def resize(self, targets: torch.Tensor | Sequence[int], *, tokens: int) -> PagePlan:
        """Move every request to its target length (int32 ``[requests]``), in one launch.

        Requests that shrink give their last pages back first; requests that grow then take
        pages, request by request and block by block, from the stack's top.  ``tokens``
        is the number of new tokens in all, or a bound on it (the plan's size).  A target
        that does not fit the block table or the stack, or more new tokens than ``tokens``,
        changes nothing, plans nothing and sets ``status_word``.
        """
        if not isinstance(targets, torch.Tensor):
            targets = torch.tensor(targets, dtype=torch.int32, device=self.device)
        if targets.dtype != torch.int32 or targets.ndim != 1 or targets.shape[0] != self.requests \
                or targets.device != self.device or not targets.is_contiguous():
            raise ValueError("targets must be a contiguous int32 vector [requests] on the cache's device")
        tokens = int(tokens)
        if not 0 <= tokens < 1 << 31:
            raise ValueError("the number of new tokens is invalid")
        requests = self.requests
        words = 4 + 4 * min(tokens, tokens // PAGE_TOKENS + 2 * requests) + requests + 1 + 2 * tokens
        self._epoch[0] += 1
        buffer = targets.new_empty(words)
        _call(self.device, "cow_pages_resize", self._at, targets.data_ptr(), tokens, buffer.data_ptr(), words)
        return PagePlan(self, self._epoch[0], tokens, buffer)

    def store(self, keys: torch.Tensor, values: torch.Tensor, plan: PagePlan, *, layer: int = 0) -> None:
        """Quantise the plan's new tokens' ``keys`` and ``values`` ``[tokens, kv_heads, head_width]`` into ``layer``.

        The scale of a page and head is the smallest power of two with ``max|x| <= 448 * scale``
        over its tokens; a page that already holds tokens keeps its scale where that is larger, and
        has its codes rounded again to a larger one.  Infinities become the largest code.
        """
        shape = (plan.tokens, self.kv_heads, self.head_width)
        if keys.shape != shape or values.shape != shape:
            raise ValueError(f"stored keys and values must be {list(shape)}")
        if plan.cache._epoch is not self._epoch or plan.epoch != self._epoch[0]:
            raise ValueError("the plan is not of this cache's last resize")
        if keys.dtype != values.dtype:
            raise ValueError("keys and values must share one dtype")
        if not 0 <= layer < self.layers:
            raise ValueError("the K/V cache has no such layer")
        (k, k0, k1), (v, v0, v1) = _rows(keys, "keys"), _rows(values, "values")
        if k.device != self.device or v.device != self.device:
            raise ValueError("keys and values must be on the cache's device")
        _call(self.device, "cow_kv8_store", self._at, layer, k.data_ptr(), k0, k1, v.data_ptr(), v0, v1, _lib.dtype_code(k.dtype), plan.buffer.data_ptr(), plan.tokens)

    def read(self, slots: torch.Tensor, *, layer: int = 0, dtype: torch.dtype = torch.bfloat16):
        """Keys and values ``[slots, kv_heads, head_width]`` that the cache holds at ``slots`` (int32; zeros for -1)."""
        if slots.dtype != torch.int32 or slots.ndim != 1 or slots.device != self.device or not slots.is_contiguous():
            raise ValueError("slots must be a contiguous int32 vector on the cache's device")
        if not 0 <= layer < self.layers:
            raise ValueError("the K/V cache has no such layer")
        code = _lib.dtype_code(dtype)
        keys, values = slots.new_empty((2, slots.shape[0], self.kv_heads, self.head_width), dtype=dtype).unbind()
        _call(self.device, "cow_kv8_read", self._at, layer, slots.data_ptr(), slots.shape[0], keys.data_ptr(),
              values.data_ptr(), code)
        return keys, values

    def attend(self, queries: torch.Tensor, *, layer: int = 0, scale: float | None = None,
               workspace: torch.Tensor | None = None) -> torch.Tensor:
        """One query token per request over its cached tokens, ``[requests, heads, head_width]``.

        ``softmax(scale * q . K) V`` with float32 sums over the ``lengths[b]`` cached tokens, ``scale`` 1 /
        sqrt(head_width) by default; zeros for a request without tokens.  16-bit queries have their weights held in
        float16, float32 ones in two of its parts.  Calls that may overlap on the GPU need a ``workspace`` each
        (``new_workspace``); the default one is made at the first call for a number of heads, which must not be
        inside a graph capture.
        """
        shape = queries.shape
        if len(shape) != 3 or shape[0] != self.requests or shape[2] != self.head_width or shape[1] < 1 or shape[1] % self.kv_heads:
            raise ValueError("attend takes queries [requests, heads, head_width], heads a multiple of kv_heads")
        if not 0 <= layer < self.layers:
            raise ValueError("the K/V cache has no such layer")
        code = _lib.dtype_code(queries.dtype)
        q, q0, q1 = _rows(queries, "queries")
        if q.device != self.device:
            raise ValueError("queries must be on the cache's device")
        heads = shape[1]
        if workspace is None:
            workspace = self._workspaces.get(heads)
            if workspace is None:
                workspace = self._workspaces[heads] = self.new_workspace(heads)
        elif workspace.dtype != torch.uint8 or workspace.device != self.device or not workspace.is_contiguous():
            raise ValueError("a workspace is a contiguous uint8 tensor on the cache's device (new_workspace)")
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        _call(self.device, "cow_kv8_attend", self._at, layer, q.data_ptr(), q0, q1, code, heads,
              self.head_width ** -0.5 if scale is None else float(scale), out.data_ptr(), workspace.data_ptr(),
              workspace.numel())
        return out

    def new_workspace(self, heads: int) -> torch.Tensor:
        """A workspace of ``attend`` for ``heads`` query heads, made outside of any graph capture."""
        _not_capturing("a workspace of attend (new_workspace)")
        need = _lib.load().cow_kv8_attend_workspace_bytes(self._at, heads)
        if need < 0:
            raise ValueError("heads must be a multiple of kv_heads")
        workspace = torch.empty(need, dtype=torch.uint8, device=self.device)
        workspace[:16].zero_()
        return workspace

    # ---- lifecycle

    def with_requests(self, keep: torch.Tensor | Sequence[int], *, new: int = 0) -> "PagedKVCache":
        """The cache with the request slots ``keep``, in their order, and ``new`` empty ones after
        them: same pages and stack.  Requests left out must have been resized to 0 (their pages
        would be lost).  The old object is not used again.  (``keep`` is checked on the host: one on the device is copied there.)"""
        try:
            keep = [operator.index(i) for i in (keep.tolist() if isinstance(keep, torch.Tensor) else keep)]
        except TypeError:
            raise ValueError("kept requests must be a vector of whole numbers") from None
        if len(set(keep)) != len(keep) or not all(0 <= i < self.requests for i in keep):
            raise ValueError(f"kept requests must be different ones of 0 .. {self.requests - 1}")
        keep = torch.tensor(keep, dtype=torch.int64, device=self.device)
        total = keep.shape[0] + new
        if new < 0 or total > MAX_REQUESTS or total * self.max_blocks >= 1 << 25:
            raise ValueError("the K/V cache exceeds the compiled limits (8192 requests, 2^25 table entries)")
        tables = self.block_tables.new_full((total, self.max_blocks), -1)
        lengths = self.lengths.new_zeros(total)
        tables[:keep.shape[0]] = self.block_tables[keep]
        lengths[:keep.shape[0]] = self.lengths[keep]
        self._epoch[0] += 1  # plans made for the old slots are over
        cache = replace(self, block_tables=tables, lengths=lengths)
        object.__setattr__(cache, "_workspaces", self._workspaces)  # their size does not depend on the requests
        return cache

    def validate_invariants(self) -> None:
        """Raise on a device error, or where live and free pages do not partition the pool (synchronises)."""
        bits = int(self.status_word.item())
        if bits:
            raise RuntimeError("; ".join(text for bit, text in _STATUS_TEXT if bits & bit) or f"K/V cache status {bits}")
        blocks = (self.lengths.long() + PAGE_TOKENS - 1) // PAGE_TOKENS
        live = torch.arange(self.max_blocks, device=self.device) < blocks[:, None]
        if bool(((self.block_tables >= 0) != live).any()):
            raise AssertionError("K/V block tables do not match the lengths")
        count = int(self.free_count.item())
        if not 0 <= count <= self.pages:
            raise AssertionError("K/V free page count is invalid")
        every = torch.cat((self.block_tables[live], self.free_pages[:count]))
        if every.numel() != self.pages or not torch.equal(every.sort().values.long(),
                                                          torch.arange(self.pages, device=self.device)):
            raise AssertionError("live and free K/V pages do not partition the cache")
