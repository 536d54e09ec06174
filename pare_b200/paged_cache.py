"""Paged KV cache held in 8 bits: block tables, append, dense reconstruction and attention for requests of any lengths.

The reference's cache (``pare/kv_cache.py:163-288``, here :class:`pare_b200.kv_cache.QuantizedKVCache`) is one dense batch whose
sequences all have the same length.  A server's requests start and end at their own times: here a pool of blocks of ``block_size``
tokens is shared by up to ``max_requests`` of them through a block table.  A block holds int8 codes with one scale per head for its
keys and one for its values; it is quantized once, when its last token arrives.  Until then the tokens stay in the input type
(``tail_k`` / ``tail_v``), so what is stored does not depend on how the tokens were cut into calls, as with the reference's
residual window.  An infinity or NaN in a block makes that head's whole block NaN once it is quantized; a query that sees one in
an open row gets no finite result.

Three functions work on plain tensors, and :class:`PagedKVCache` keeps those tensors for all layers of a model:

* :func:`plan_blocks` makes the tables of a step on the GPU from the requests' lengths: which rows belong to whom, where each new
  token goes, which blocks are taken.  One step serves every layer.
* :func:`append_blocks` stores a step's new keys and values in one layer, :func:`dense_blocks` gives whole sequences back.
* :func:`attend_blocks` is the attention of the step's queries over the layer: one new token per request (decode) or several
  (short prompts, continuations), causal by position.

A step's tokens stay: there is no way to take some of them back (drafted tokens that turn out wrong, say), for a block that they
filled up has been quantized with them, and its open rows hold the tokens behind it.  And attention reads what is stored: where a block
fills up inside a step, the step's earlier tokens see their own block in 8 bits too, with a scale that the later ones had a part in (an
infinity among those reaches them).  Fed one by one they would have seen it in 16 bits.

Nothing here computes gradients, and everything runs on CUDA tensors only.
"""

from __future__ import annotations

import ctypes
import functools
import math
import threading
from dataclasses import dataclass
from typing import NamedTuple, Sequence

import torch
from torch import Tensor

from pare_b200.kernels import _lib
from pare_b200.kv_cache import prefill_attention

BLOCK_SIZES = (16, 32, 64)
HEAD_DIMS = (64, 128)
MAX_REQUESTS = 4096
MAX_QUERY_TOKENS = 4096      # rows of a step that attend_blocks takes
_REFUSED = {1: "a length or number of new tokens is negative", 2: "more new tokens than rows",
            4: "a request would not fit its row of the block table", 8: "not enough free blocks"}


class _LayerTensors(NamedTuple):
    k_codes: Tensor
    v_codes: Tensor
    k_scale: Tensor
    v_scale: Tensor
    tail_k: Tensor
    tail_v: Tensor


class PagedLayer(_LayerTensors):
    """One layer's storage, ``PagedLayer(k_codes, v_codes, k_scale, v_scale, tail_k, tail_v)``: codes int8
    ``[num_blocks, H, block_size, D]``, scales float32 ``[num_blocks, H]`` (value = code * scale), open blocks' tokens float16 /
    bfloat16 ``[requests, H, block_size, D]``, all contiguous on one device.  Checked once, here; the tensors stay where they are."""

    def __new__(cls, *tensors: Tensor, **named: Tensor) -> "PagedLayer":
        self = super().__new__(cls, *tensors, **named)
        codes = self.k_codes
        if codes.dim() != 4 or self.tail_k.dim() != 4:
            raise ValueError("paged layer: codes [num_blocks, heads, block_size, head_dim], open rows [requests, heads, block_size, head_dim]")
        (n, h, bs, d), requests, dtype, device = codes.shape, self.tail_k.shape[0], self.tail_k.dtype, codes.device
        if bs not in BLOCK_SIZES or d not in HEAD_DIMS or dtype not in (torch.float16, torch.bfloat16) or n < 1 or h < 1 or requests < 1:
            raise ValueError(f"paged layer: {n} blocks of {bs} tokens (one of {BLOCK_SIZES}), {h} heads of {d} channels (one of {HEAD_DIMS}), "
                             f"{requests} requests, open rows in {dtype}")
        if device.type != "cuda":
            raise RuntimeError("paged layers are CUDA tensors")
        for t, shape, want in zip(self, ((n, h, bs, d),) * 2 + ((n, h),) * 2 + ((requests, h, bs, d),) * 2,
                                  (torch.int8,) * 2 + (torch.float32,) * 2 + (dtype,) * 2):
            if t.shape != shape or t.dtype is not want or t.device != device or not t.is_contiguous() or t.data_ptr() % 16:
                raise ValueError(f"paged layer: expected a contiguous, 16-byte aligned {want} tensor {list(shape)} on {device}, got {t.dtype} "
                                 f"{list(t.shape)} on {t.device}")
        self.num_blocks, self.heads, self.block_size, self.head_dim, self.requests = n, h, bs, d, requests
        self.dtype, self.device = dtype, device
        self._struct = _lib.PagedLayerStruct(*(t.data_ptr() for t in self), n, requests, h, bs, d, _lib.dtype_code(dtype))
        self._c = ctypes.addressof(self._struct)
        return self

    # Copies and other tensors in a layer's place are layers of their own, with their own addresses.
    @classmethod
    def _make(cls, tensors) -> "PagedLayer":
        return cls(*tensors)

    def __reduce__(self):
        return PagedLayer, tuple(self)


_first_use = threading.Lock()


@functools.lru_cache(maxsize=4096)
def _step_layout(requests: int, tokens: int, block_size: int) -> tuple[int, tuple[int, ...]]:
    """Bytes of a step, and the offset of each of its fields in 32-bit words."""
    L = _lib.lib()
    nbytes = L.pare_paged_step_bytes(requests, tokens, block_size)
    if nbytes == 0:
        raise ValueError(f"plan_blocks: {requests} requests (at most {MAX_REQUESTS}), {tokens} rows, blocks of {block_size} (one of {BLOCK_SIZES})")
    return nbytes, tuple(L.pare_paged_step_offset(f, requests, tokens, block_size) // 4 for f in range(7))


class PagedStep:
    """Tables of one step (made by :func:`plan_blocks`); the properties are views of one buffer on the GPU."""

    __slots__ = ("words", "requests", "tokens", "block_size", "block_table", "device", "lengths", "written_once", "_at", "_ld", "_struct", "_c")

    def __init__(self, words: Tensor, at: tuple[int, ...], requests: int, tokens: int, block_size: int, block_table: Tensor, ld: int) -> None:
        self.words, self._at, self.device = words, at, words.device
        self.requests, self.tokens, self.block_size, self.block_table, self._ld = requests, tokens, block_size, block_table, ld
        self.lengths: list[tuple[int, int]] | None = None    # (old, new) per request where the host knows them
        self.written_once = False      # True: no graph writes the step again, so lengths that were read from it stay true
        self._c = 0

    def _tables(self) -> int:
        """Address of the step as the C entries take it."""
        if not self._c:
            with _first_use:       # threads may share a step
                if not self._c:
                    self._struct = _lib.PagedTablesStruct(self.words.data_ptr(), self.block_table.data_ptr(), self._ld, self.block_table.shape[1],
                                                          self.requests, self.tokens, self.block_size)
                    self._c = ctypes.addressof(self._struct)
        return self._c

    @property
    def query_start(self) -> Tensor:
        """int32 ``[requests + 1]``: first row of each request's new tokens."""
        return self.words.as_strided((self.requests + 1,), (1,), self._at[1])

    @property
    def seq_lens(self) -> Tensor:
        """int32 ``[requests]``: lengths after the step."""
        return self.words.as_strided((self.requests,), (1,), self._at[2])

    @property
    def free_count(self) -> Tensor:
        """int32 ``[1]``: free blocks after the step."""
        return self.words.as_strided((1,), (1,), self._at[2] + self.requests)

    @property
    def context_start(self) -> Tensor:
        """int64 ``[requests + 1]``: first row of each request in :func:`dense_blocks`' result."""
        return self.words.as_strided((2 * (self.requests + 1),), (1,), self._at[3]).view(torch.int64)

    @property
    def slots(self) -> Tensor:
        """int64 ``[tokens]``: ``block id * block_size + offset`` of each row, -1 for rows that belong to nobody."""
        return self.words.as_strided((2 * self.tokens,), (1,), self._at[4]).view(torch.int64)

    @property
    def token_request(self) -> Tensor:
        """int32 ``[tokens]``: request of each row, -1 for nobody."""
        return self.words.as_strided((self.tokens,), (1,), self._at[5])

    @property
    def positions(self) -> Tensor:
        """int32 ``[tokens]``: position of each row in its request, -1 for rows that belong to nobody."""
        return self.words.as_strided((self.tokens,), (1,), self._at[6])

    def check(self) -> None:
        """Raise if the step was refused (waits for the GPU)."""
        status = int(self.words[0])
        if status:
            raise RuntimeError("paged step refused: " + ", ".join(t for bit, t in _REFUSED.items() if status & bit))


def _call(device: torch.device, fn, what: str, *args) -> None:
    """``fn(*args, stream)`` on ``device``, whichever device is current."""
    if device.index == _lib.current_device():
        status = fn(*args, _lib.current_stream(device))
    else:
        with torch.cuda.device(device):
            status = fn(*args, _lib.current_stream(device))
    if status:
        _lib.check(status, what)


def _ints(t: Tensor, shape: tuple, device, what: str) -> None:
    if t.dtype is not torch.int32 or t.shape != shape or t.device != device or not t.is_contiguous():
        raise ValueError(f"{what} must be a contiguous int32 tensor {list(shape)} on {device}, got {t.dtype} {list(t.shape)} on {t.device}")


def plan_blocks(seq_lens: Tensor, new_lens: Tensor, block_table: Tensor, free_blocks: Tensor, free_count: Tensor, block_size: int,
                tokens: int) -> PagedStep:
    """Tables of a step in which request ``r`` gets ``new_lens[r]`` more tokens on top of ``seq_lens[r]``.

    ``seq_lens``, ``new_lens`` int32 ``[requests]``; ``block_table`` int32 ``[requests, blocks per request]``, updated in place with
    the blocks that the step takes from the top of the stack ``free_blocks`` (int32; ``free_count`` int32 ``[1]`` of them).  The
    new tokens lie one request after the other over ``tokens`` rows; rows behind them belong to nobody (a padded batch).  All
    lengths stay on the GPU: nothing waits for it.  A step that does not fit is refused as a whole (no row belongs to anybody,
    lengths and free blocks stay): :meth:`PagedStep.check`.  Other inputs than the table are not written; to go on from the step,
    use its ``seq_lens`` and ``free_count``.
    """
    dev, index, i32 = seq_lens.device, seq_lens.get_device(), torch.int32
    if dev.type != "cuda":
        raise RuntimeError("plan_blocks runs on CUDA tensors only")
    n, capacity = seq_lens.numel(), free_blocks.numel()
    width = ld = block_table.shape[1] if block_table.dim() == 2 else 0
    if not (seq_lens.dtype is new_lens.dtype is free_blocks.dtype is free_count.dtype is block_table.dtype is i32
            and seq_lens.dim() == new_lens.dim() == free_blocks.dim() == free_count.dim() == 1 and new_lens.numel() == n and free_count.numel() == 1
            and width and block_table.shape[0] == n
            and index == new_lens.get_device() == free_blocks.get_device() == free_count.get_device() == block_table.get_device()
            and seq_lens.is_contiguous() and new_lens.is_contiguous() and free_blocks.is_contiguous() and free_count.is_contiguous()
            and block_table.is_contiguous()):
        for t, want, what in ((seq_lens, (n,), "seq_lens"), (new_lens, (n,), "new_lens"), (free_count, (1,), "free_count"),
                              (free_blocks, (capacity,), "free_blocks")):
            _ints(t, want, dev, what)
        if (block_table.dtype is not i32 or not width or block_table.shape[0] != n or block_table.device != dev or block_table.stride(1) != 1
                or (n > 1 and block_table.stride(0) < width)):
            raise ValueError(f"block_table must be int32 [{n}, blocks per request] with adjacent columns on {dev}")
        ld = block_table.stride(0) if n > 1 else width
    nbytes, at = _step_layout(n, tokens, block_size)
    words = seq_lens.new_empty(nbytes // 4)
    step = PagedStep(words, at, n, tokens, block_size, block_table, ld)
    _call(dev, _lib.lib().pare_paged_plan, "pare_paged_plan", seq_lens.data_ptr(), new_lens.data_ptr(), n, block_table.data_ptr(),
          ld, width, free_blocks.data_ptr(), capacity, free_count.data_ptr(), block_size, tokens, words.data_ptr(), nbytes)
    return step


def _fits(layer: PagedLayer, step: PagedStep) -> None:
    if layer.block_size != step.block_size or layer.requests != step.requests or layer.device != step.device:
        raise ValueError(f"the layer ({layer.requests} requests, blocks of {layer.block_size}, {layer.device}) and the step ({step.requests}, "
                         f"{step.block_size}, {step.device}) do not belong together")


def _rows(t: Tensor, tokens: int, heads: int, layer: PagedLayer, what: str) -> tuple[Tensor, int, int, int]:
    """A step's rows as the kernels take them (channels adjacent, 16-byte aligned rows), their address and strides."""
    if t.shape != (tokens, heads, layer.head_dim) or t.dtype is not layer.dtype or t.device != layer.device:
        raise ValueError(f"{what} must be {layer.dtype} {[tokens, heads, layer.head_dim]} on {layer.device}, got {t.dtype} {list(t.shape)} on {t.device}")
    (a, b, c), p = t.stride(), t.data_ptr()
    if c == 1 and not (a | b) & 7 and not p & 15:
        return t, p, a, b
    t = t.clone(memory_format=torch.contiguous_format)
    return t, t.data_ptr(), t.stride(0), t.stride(1)


def append_blocks(layer: PagedLayer, step: PagedStep, k: Tensor, v: Tensor) -> None:
    """Store the step's new keys and values ``[tokens, H, D]`` in one layer: blocks that fill up are quantized into the pool, the
    rest goes to the open rows.  Once per step and layer: a block that filled up had its open rows written over by the tokens behind it,
    so the same call again would quantize it from those."""
    _fits(layer, step)
    tokens, heads, dev = step.tokens, layer.heads, layer.device
    k, kp, kt, kh = _rows(k, tokens, heads, layer, "k")
    v, vp, vt, vh = _rows(v, tokens, heads, layer, "v")
    if dev.index != _lib.current_device():
        with torch.cuda.device(dev):
            return append_blocks(layer, step, k, v)
    status = _lib.lib().pare_paged_append(kp, vp, kt, kh, vt, vh, layer._c, step._c or step._tables(), _lib.current_stream(dev))
    if status:
        _lib.check(status, "pare_paged_append")


def dense_blocks(layer: PagedLayer, step: PagedStep, total: int) -> tuple[Tensor, Tensor]:
    """Keys and values, after the step's append, of every request with new tokens in it: two tensors ``[total, H, D]`` of the open
    rows' dtype, request ``r`` from row ``step.context_start[r]`` on (``total``: the sum of those requests' lengths; rows beyond it
    are left out, rows behind the last token are zeros)."""
    _fits(layer, step)
    k = layer.tail_k.new_empty(total, layer.heads, layer.head_dim)
    v = torch.empty_like(k)
    _call(layer.device, _lib.lib().pare_paged_dense, "pare_paged_dense", layer._c, step._tables(), k.data_ptr(), v.data_ptr(), total)
    return k, v


@functools.lru_cache(maxsize=64)
def _attn_workspace(d: int, index: int) -> int:
    with torch.cuda.device(index):
        return _lib.lib().pare_paged_attn_workspace_bytes(d)


def attend_blocks(layer: PagedLayer, step: PagedStep, q: Tensor, scale: float | None = None, out: Tensor | None = None) -> Tensor:
    """``softmax(q K^T * scale) V`` of the step's queries ``q [tokens, Hq, D]`` over their request's tokens up to and with their own
    (the step's keys and values have been appended).  ``Hq`` is a multiple of the KV heads; default scale ``1 / sqrt(D)``.  At most
    4096 rows: longer prompts go through :meth:`PagedKVCache.prefill` (and rows times tokens of a full row of the block table stay
    below 2^35).  Rows that belong to nobody are left as they were in
    ``out`` (``[tokens, Hq, D]``, channels adjacent, not overlapping ``q``; a new tensor, with anything in those rows, if not given)."""
    return _attend(layer, step, q, None, None, scale, out)


def _attend(layer: PagedLayer, step: PagedStep, q: Tensor, new_k: Tensor | None, new_v: Tensor | None, scale: float | None, out: Tensor | None) -> Tensor:
    """:func:`attend_blocks`, where ``new_k`` is given after :func:`append_blocks`: what is refused has not been stored either."""
    _fits(layer, step)
    tokens, d, dev = step.tokens, layer.head_dim, layer.device
    hq = q.size(1) if q.dim() == 3 else 0
    if hq == 0 or hq % layer.heads:
        raise ValueError(f"attend_blocks: q [tokens, heads, {d}] with a multiple of {layer.heads} heads, got {list(q.shape)}")
    if tokens > MAX_QUERY_TOKENS:
        raise ValueError(f"attend_blocks takes at most {MAX_QUERY_TOKENS} rows, got {tokens}")
    if tokens > 15 and tokens * (step.block_table.shape[1] * step.block_size // 16 + 2) >= 1 << 31:      # a row of the table has less than 2^31 tokens
        raise ValueError(f"attend_blocks: {tokens} rows times {step.block_table.shape[1]} blocks of {step.block_size} tokens a request are too many to count")
    q, qp, qt, qh = _rows(q, tokens, hq, layer, "q")
    if out is None:
        out = q.new_empty(tokens, hq, d)
        ot, oh = hq * d, d
    elif out.shape != q.shape or out.dtype is not q.dtype or out.device != dev or out.stride(2) != 1:
        raise ValueError(f"out must be {q.dtype} {list(q.shape)} on {dev} with adjacent channels")
    else:
        ot, oh, _ = out.stride()
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    if dev.index != _lib.current_device():
        with torch.cuda.device(dev):
            return _attend(layer, step, q, new_k, new_v, scale, out)
    stream, nbytes = _lib.current_stream(dev), _attn_workspace(d, dev.index)
    ws = _lib.scratch(dev, nbytes, stream)
    if new_k is not None:
        append_blocks(layer, step, new_k, new_v)
    status = _lib.lib().pare_paged_attn(qp, qt, qh, layer._c, step._c or step._tables(), hq, out.data_ptr(), ot, oh, scale, ws.data_ptr(), nbytes, stream)
    if status:
        _lib.check(status, "pare_paged_attn")
    return out


@dataclass
class PagedKVConfig:
    """``num_blocks`` blocks of ``block_size`` (16, 32 or 64) tokens in the pool, up to ``max_requests`` requests of up to
    ``max_seq_len`` tokens (to the end of the last block where the GPU alone knows the lengths)."""

    num_blocks: int
    block_size: int = 32
    max_requests: int = 64
    max_seq_len: int = 8192


class PagedKVCache:
    """Paged 8-bit KV cache of a model: one pool per layer, tables shared by all layers.

    Requests are numbered ``0 .. max_requests - 1``.  A step: :meth:`plan` with the number of new tokens of every request, then for
    each layer :meth:`attend` (decode) or :meth:`prefill` (prompts) with the step's queries, keys and values ``[tokens, heads, D]``,
    the requests' tokens one after the other.  :meth:`release` ends requests.  Calls on one cache belong on one stream.
    """

    def __init__(self, num_layers: int, num_kv_heads: int, head_dim: int, config: PagedKVConfig, dtype: torch.dtype = torch.bfloat16,
                 device="cuda") -> None:
        c = config
        if c.block_size not in BLOCK_SIZES or head_dim not in HEAD_DIMS or dtype not in (torch.float16, torch.bfloat16):
            raise ValueError(f"PagedKVCache: block_size one of {BLOCK_SIZES}, head_dim one of {HEAD_DIMS}, float16 or bfloat16")
        if not 1 <= c.max_requests <= MAX_REQUESTS or c.num_blocks < 1 or c.max_seq_len < 1 or num_kv_heads < 1:
            raise ValueError(f"PagedKVCache: 1 to {MAX_REQUESTS} requests, at least one block, token and head")
        device = torch.device(device)
        if device.type != "cuda":
            raise RuntimeError("PagedKVCache runs on CUDA tensors only (no CPU implementation).")
        if device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        self.num_layers, self.config, self.dtype, self.device = num_layers, c, dtype, device
        codes, scale, tail = ((c.num_blocks, num_kv_heads, c.block_size, head_dim), (c.num_blocks, num_kv_heads),
                              (c.max_requests, num_kv_heads, c.block_size, head_dim))
        self.layers = [PagedLayer(*(torch.empty(codes, dtype=torch.int8, device=device) for _ in range(2)),
                                  *(torch.zeros(scale, dtype=torch.float32, device=device) for _ in range(2)),
                                  *(torch.zeros(tail, dtype=dtype, device=device) for _ in range(2))) for _ in range(num_layers)]
        self.block_table = torch.zeros(c.max_requests, -(-c.max_seq_len // c.block_size), dtype=torch.int32, device=device)
        self._state = torch.zeros(c.max_requests + 1, dtype=torch.int32, device=device)    # lengths, then the number of free blocks
        self.seq_lens, self.free_count = self._state[:-1], self._state[-1:]
        self.free_blocks = torch.empty(c.num_blocks, dtype=torch.int32, device=device)
        self._captured = False      # a graph changes the lengths: the host cannot follow them any more
        self.reset()

    def reset(self) -> None:
        """Forget every request."""
        c = self.config
        self.free_blocks.copy_(torch.arange(c.num_blocks - 1, -1, -1, dtype=torch.int32))
        self._state.zero_()
        self._state[-1] = c.num_blocks
        self._lens: list[int] | None = None if self._captured else [0] * c.max_requests       # None: lengths are known to the GPU alone

    # ------------------------------------------------------------------ lengths
    def _blocks(self, n: int) -> int:
        return -(-n // self.config.block_size)

    def seq_len(self, request: int) -> int:
        """Tokens of a request (waits for the GPU if lengths have been given as a tensor)."""
        return self._lens[request] if self._lens is not None else int(self.seq_lens[request])

    def free_block_count(self) -> int:
        return self.config.num_blocks - sum(map(self._blocks, self._lens)) if self._lens is not None else int(self.free_count)

    def plan(self, new_lens: Sequence[int] | dict[int, int] | Tensor, tokens: int | None = None) -> PagedStep:
        """Begin a step: ``new_lens`` new tokens per request -- a sequence over all requests, a dict ``{request: tokens}``, or an
        int32 tensor ``[max_requests]`` on the GPU (then ``tokens``, the number of rows, is needed, the host learns of no
        lengths, and a step that does not fit is refused by the GPU: :meth:`PagedStep.check`).  Numbers that the host knows are
        checked here.  ``tokens`` may be larger than the sum (a padded batch)."""
        c, lengths = self.config, None
        if isinstance(new_lens, Tensor):
            if tokens is None:
                raise ValueError("plan: the number of rows is needed when lengths are on the GPU")
            captured = torch.cuda.is_current_stream_capturing()
            self._captured |= captured
        else:
            captured = False      # a copy from the host cannot be captured
            if isinstance(new_lens, dict):
                if any(not 0 <= r < c.max_requests for r in new_lens):
                    raise ValueError(f"plan: requests are numbered 0 to {c.max_requests - 1}")
                new = [new_lens.get(r, 0) for r in range(c.max_requests)]
            else:
                new = list(new_lens)
                if len(new) != c.max_requests:
                    raise ValueError(f"plan: a number for each of the {c.max_requests} requests, got {len(new)}")
            if any(n < 0 for n in new):
                raise ValueError("plan: negative number of tokens")
            total = sum(new)
            tokens = total if tokens is None else tokens
            if tokens < total:
                raise ValueError(f"plan: {total} new tokens over {tokens} rows")
            if self._lens is not None:
                end = [a + n for a, n in zip(self._lens, new)]
                if max(end) > c.max_seq_len:
                    raise ValueError(f"plan: request {end.index(max(end))} would have {max(end)} tokens (at most {c.max_seq_len})")
                if sum(map(self._blocks, end)) > c.num_blocks:
                    raise RuntimeError(f"plan: {sum(map(self._blocks, end))} blocks needed, {c.num_blocks} in the pool")
                lengths = list(zip(self._lens, new))
            new_lens = torch.tensor(new, dtype=torch.int32).to(self.device)
        step = plan_blocks(self.seq_lens, new_lens, self.block_table, self.free_blocks, self.free_count, c.block_size, tokens)
        self._state.copy_(step.words.narrow(0, step._at[2], c.max_requests + 1))
        step.lengths, step.written_once = lengths, not captured
        self._lens = None if lengths is None else [a + n for a, n in lengths]
        return step

    def release(self, requests: Sequence[int] | Tensor) -> None:
        """End requests: their blocks become free and their lengths 0.  A sequence of numbers, or an int32 tensor
        ``[max_requests]`` on the GPU with a 1 for each that ends."""
        c = self.config
        if isinstance(requests, Tensor):
            mask = requests
            _ints(mask, (c.max_requests,), self.device, "release")
            self._captured |= torch.cuda.is_current_stream_capturing()
            self._lens = None
        else:
            ending = set(requests)
            if any(not 0 <= r < c.max_requests for r in ending):
                raise ValueError(f"release: requests are numbered 0 to {c.max_requests - 1}")
            mask = torch.tensor([int(r in ending) for r in range(c.max_requests)], dtype=torch.int32).to(self.device)
            if self._lens is not None:
                self._lens = [0 if r in ending else n for r, n in enumerate(self._lens)]
        table = self.block_table
        _call(self.device, _lib.lib().pare_paged_release, "pare_paged_release", mask.data_ptr(), self.seq_lens.data_ptr(), c.max_requests,
              table.data_ptr(), table.stride(0), table.shape[1], self.free_blocks.data_ptr(), c.num_blocks, self.free_count.data_ptr(),
              c.block_size)

    # ------------------------------------------------------------------ a layer's part of a step
    def append(self, layer_idx: int, step: PagedStep, new_k: Tensor, new_v: Tensor) -> None:
        """Store the step's keys and values ``[tokens, H, D]`` in a layer."""
        append_blocks(self.layers[layer_idx], step, new_k, new_v)

    def attend(self, layer_idx: int, step: PagedStep, q: Tensor, new_k: Tensor, new_v: Tensor, scale: float | None = None,
               out: Tensor | None = None) -> Tensor:
        """Append the step's keys and values, then attention of its queries over the whole requests (:func:`attend_blocks`).  Once per
        step and layer; a call that is refused has stored nothing."""
        if new_k is None:
            raise ValueError("attend: the step's keys and values are needed")
        return _attend(self.layers[layer_idx], step, q, new_k, new_v, scale, out)

    def prefill(self, layer_idx: int, step: PagedStep, q: Tensor, new_k: Tensor, new_v: Tensor, scale: float | None = None) -> Tensor:
        """Causal attention of prompts' queries ``[tokens, Hq, D]`` with the step's own keys and values at full precision, older
        tokens as the cache holds them, and the append (``head_dim`` 128; what ``QuantizedKVCache.prefill`` does, request by
        request on the prompt attention kernel).  The host needs the lengths: where they were given as tensors it waits for
        them, once for a step of :meth:`plan`, but in every call where a graph that may have been replayed since, or
        :func:`plan_blocks`, made it.  Rows behind the last token hold anything.  Once per step and layer; a call that is refused has stored nothing."""
        layer = self.layers[layer_idx]
        if layer.head_dim != 128:
            raise ValueError("prefill needs head_dim 128: use attend")
        _fits(layer, step)
        hq = q.shape[1] if q.dim() == 3 else 0
        q = _rows(q, step.tokens, hq, layer, "q")[0]
        if hq == 0 or hq % layer.heads:
            raise ValueError(f"prefill: q [tokens, heads, {layer.head_dim}] with a multiple of {layer.heads} heads, got {list(q.shape)}")
        scale = None if scale is None else float(scale)
        lengths = step.lengths
        if lengths is None:
            step.check()
            start, end = step.query_start.tolist(), step.seq_lens.tolist()
            lengths = [(e - (b - a), b - a) for e, a, b in zip(end, start, start[1:])]
            if step.written_once:
                step.lengths = lengths
        append_blocks(layer, step, new_k, new_v)
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        full_k = full_v = None
        if any(old and new for old, new in lengths):
            full_k, full_v = dense_blocks(layer, step, sum(old + new for old, new in lengths if new))
        row = ctx = 0
        with torch.cuda.device(self.device):
            for old, new in lengths:
                if not new:
                    continue
                k, v = new_k[row:row + new], new_v[row:row + new]
                if old:
                    full_k[ctx + old:ctx + old + new] = k
                    full_v[ctx + old:ctx + old + new] = v
                    k, v = full_k[ctx:ctx + old + new], full_v[ctx:ctx + old + new]
                out[row:row + new] = prefill_attention(*(t.unsqueeze(0).transpose(1, 2) for t in (q[row:row + new], k, v)), scale)[0].transpose(0, 1)
                row += new
                ctx += old + new
        return out

    def memory_bytes(self) -> dict[str, int]:
        """Bytes of the pools, of the open rows and of both, over all layers (what is allocated, whoever uses it)."""
        pool = sum(t.numel() * t.element_size() for layer in self.layers for t in layer[:4])
        rows = sum(t.numel() * t.element_size() for layer in self.layers for t in layer[4:])
        return {"blocks": pool, "open": rows, "total": pool + rows}
