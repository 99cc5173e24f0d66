"""A KV cache in 8 bits that grows while it is decoded from.

The reference's quantized segments (unicache/storage/physical.py:204-332) are
frozen when they are built; this cache is written row by row or prompt by
prompt and read by the next launch.  Keys and values lie in blocks of a pool
that a table assigns to sequences, one fp32 scale for each block and KV head,
and the smallest and largest key code of each channel of a block bound its
logits, so that a query can name the blocks it needs before it reads them.
Lengths and table are device tensors: a step over the cache can be captured as
a CUDA graph, and all layers of a model share them.
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass

import torch

from .. import _capi, kernels
from .physical import tensor_bytes

BLOCK_SIZES = (16, 32, 64, 128)


@dataclass(frozen=True, eq=False)
class Int8BlockCache:
    """8-bit keys and values of several sequences (value = code * scale).

    A block's scale is max(amax / 127, 2^-120) over its tokens so far and all
    channels of one head, a code clamp(rint(x * (1 / scale)), -127, 127).  The
    unquantised rows of the last block that a write touched stay in
    ``pending_key`` / ``pending_value``: after each write of a sequence's rows it is, bit for
    bit, the quantisation of those that count, whatever the portions in
    which they came and whatever was withdrawn (``advance``) between them.  A NaN or an infinity poisons its block (the scale becomes NaN or
    infinite), so it shows in the attention's output.

    ``lengths`` counts the tokens of each sequence and is advanced by the caller
    before a write (``advance``), once for all layers that share it.
    """

    key_code: torch.Tensor       # int8 [blocks, kv_heads, block_size, head_dim]
    key_scale: torch.Tensor      # float32 [blocks, kv_heads]
    key_low: torch.Tensor        # int8 [blocks, kv_heads, head_dim]
    key_high: torch.Tensor
    value_code: torch.Tensor
    value_scale: torch.Tensor
    pending_key: torch.Tensor    # bf16 or f16 [num_seqs, kv_heads, block_size, head_dim]
    pending_value: torch.Tensor
    block_table: torch.Tensor    # int32 [num_seqs, max_blocks]
    lengths: torch.Tensor        # int32 [num_seqs]

    def __post_init__(self):
        kernels.require_cuda(self.key_code, "key_code")
        if self.key_code.dim() != 4 or self.block_table.dim() != 2:
            raise ValueError("key_code must be [blocks, kv_heads, block_size, head_dim], block_table [num_seqs, max_blocks]")
        blocks, heads, size, dim = map(int, self.key_code.shape)
        seqs, width = map(int, self.block_table.shape)
        if size not in BLOCK_SIZES or dim not in (64, 128):
            raise ValueError(f"the block cache takes head_dim 64 or 128 and block sizes {BLOCK_SIZES}")
        if not 1 <= seqs <= 4096 or blocks < 1 or heads < 1 or width < 1:
            raise ValueError("the block cache needs 1 to 4096 sequences and at least one block and head")
        if self.pending_key.dtype not in (torch.bfloat16, torch.float16):
            raise ValueError("the block cache takes bfloat16 or float16 rows")
        rows, pending = (blocks, heads, size, dim), (seqs, heads, size, dim)
        for name, shape, dtype in (
                ("key_code", rows, torch.int8), ("value_code", rows, torch.int8),
                ("key_scale", (blocks, heads), torch.float32), ("value_scale", (blocks, heads), torch.float32),
                ("key_low", (blocks, heads, dim), torch.int8), ("key_high", (blocks, heads, dim), torch.int8),
                ("pending_key", pending, self.pending_key.dtype), ("pending_value", pending, self.pending_key.dtype),
                ("block_table", (seqs, width), torch.int32), ("lengths", (seqs,), torch.int32)):
            tensor = getattr(self, name)
            if tuple(tensor.shape) != shape or tensor.dtype != dtype or tensor.device != self.key_code.device \
                    or not tensor.is_contiguous():
                raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {shape} on the cache's device")
        struct = _capi.UcbBlock8Cache(
            key_code=self.key_code.data_ptr(), value_code=self.value_code.data_ptr(),
            key_scale=self.key_scale.data_ptr(), value_scale=self.value_scale.data_ptr(),
            key_low=self.key_low.data_ptr(), key_high=self.key_high.data_ptr(),
            pending_key=self.pending_key.data_ptr(), pending_value=self.pending_value.data_ptr(),
            block_table=self.block_table.data_ptr(), lengths=self.lengths.data_ptr(), num_blocks=blocks,
            num_seqs=seqs, max_blocks=width, kv_heads=heads, head_dim=dim, block_tokens=size,
            dtype=kernels.dtype_code(self.pending_key.dtype))
        # the launch wrappers read these on every call
        for name, attribute in (("_struct", struct), ("descriptor", ctypes.addressof(struct)),
                                ("device", self.key_code.device), ("index", self.key_code.get_device()),
                                ("dtype", self.pending_key.dtype),
                                ("num_seqs", seqs), ("num_kv_heads", heads), ("head_dim", dim),
                                ("block_size", size), ("max_tokens", width * size), ("_workspace_bytes", {}), ("_shapes", {})):
            object.__setattr__(self, name, attribute)
        lib = _capi.load()
        object.__setattr__(self, "select_bytes", int(lib.ucb_block8_select_workspace_bytes(self.descriptor)))
        if self.select_bytes < 0:
            _capi.check(_capi.UCB_ERR_INVALID, "Int8BlockCache")

    @classmethod
    def allocate(cls, num_seqs: int, max_tokens: int, *, num_kv_heads: int, head_dim: int = 128, block_size: int = 64,
                 dtype: torch.dtype = torch.bfloat16, device: torch.device | str = "cuda",
                 block_table: torch.Tensor | None = None, num_blocks: int | None = None,
                 lengths: torch.Tensor | None = None) -> "Int8BlockCache":
        """An empty cache of ``num_seqs`` sequences of up to ``max_tokens``
        tokens.  ``block_table`` (int32 [num_seqs, max_blocks], with the pool's
        ``num_blocks``) and ``lengths`` may be those of another cache, as the layers of one model
        share them; without a table every sequence has its own consecutive blocks."""

        device = torch.device(device)
        if device.type != "cuda":
            raise RuntimeError("the block cache lives on a CUDA device: the b200 backend has no CPU path")
        if device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        if num_seqs < 1 or max_tokens < 1 or block_size not in BLOCK_SIZES:
            raise ValueError(f"need num_seqs and max_tokens of at least 1 and a block size of {BLOCK_SIZES}")
        width = -(-max_tokens // block_size)
        if block_table is None:
            if num_blocks is not None and num_blocks < num_seqs * width:
                raise ValueError("without a block_table the pool needs a block for every table entry")
            block_table = torch.arange(num_seqs * width, device=device, dtype=torch.int32).view(num_seqs, width)
            num_blocks = num_blocks or num_seqs * width
        elif num_blocks is None:
            raise ValueError("a given block_table needs num_blocks")
        if lengths is None:
            lengths = torch.zeros(num_seqs, device=device, dtype=torch.int32)
        rows = (num_blocks, num_kv_heads, block_size, head_dim)

        def zeros(shape, kind):
            return torch.zeros(shape, device=device, dtype=kind)

        return cls(key_code=zeros(rows, torch.int8), key_scale=zeros(rows[:2], torch.float32),
                   key_low=zeros((num_blocks, num_kv_heads, head_dim), torch.int8),
                   key_high=zeros((num_blocks, num_kv_heads, head_dim), torch.int8),
                   value_code=zeros(rows, torch.int8), value_scale=zeros(rows[:2], torch.float32),
                   pending_key=zeros((num_seqs, *rows[1:]), dtype), pending_value=zeros((num_seqs, *rows[1:]), dtype),
                   block_table=block_table, lengths=lengths)

    @classmethod
    def from_dense(cls, keys: list, values: list, *, max_tokens: int | None = None,
                   block_size: int = 64) -> "Int8BlockCache":
        """A cache of the sequences whose keys and values [T_i, H, D] are given,
        with room for ``max_tokens`` tokens each (default: the longest)."""

        if not keys or len(keys) != len(values):
            raise ValueError("from_dense needs matching, non-empty key and value lists")
        for key, value in zip(keys, values):
            if key.dim() != 3 or key.shape != value.shape:
                raise ValueError("the block cache expects matching [tokens, kv_heads, head_dim] tensors")
            kernels.require_cuda(key, "key")
        counts = [int(k.shape[0]) for k in keys]
        if max_tokens is not None and max_tokens < max(counts):
            raise ValueError("max_tokens is below the longest sequence")
        cache = cls.allocate(len(keys), max(1, *counts, max_tokens or 1), num_kv_heads=int(keys[0].shape[1]),
                             head_dim=int(keys[0].shape[2]), block_size=block_size, dtype=keys[0].dtype,
                             device=keys[0].device)
        starts = torch.tensor([0, *counts], dtype=torch.int32).cumsum(0, dtype=torch.int32).to(cache.device)
        cache.advance(starts[1:] - starts[:-1])
        cache.write(torch.cat(keys), torch.cat(values), starts=starts)
        return cache

    # ---------------------------------------------------------------- use
    def advance(self, tokens) -> None:
        """Add ``tokens`` (a number or an int32 [num_seqs] tensor) to the lengths
        before the write of that many rows: once for all caches that share them.  Over a
        ``BlockPool`` its ``advance`` takes the place of this one.

        Negative numbers withdraw the last rows, such as rejected drafts: as far as the start of
        the last block written, or back to the end of an earlier block.  From the middle
        of an earlier block on there is no way forward: its unquantised rows are gone, and a write
        there is refused (device error bit 2).  So a draft that may be rejected in part ends with
        its block at the latest."""

        self.lengths.add_(tokens)

    def write(self, key: torch.Tensor, value: torch.Tensor, *, starts: torch.Tensor | None = None) -> None:
        """Rows [N, kv_heads, head_dim] become the last tokens of the sequences:
        rows ``starts[s]`` to ``starts[s + 1]`` (int32 [num_seqs + 1] on the
        device) of sequence s, or one row each without ``starts``.  ``lengths`` already
        counts them.  Sequences with a length past the table or malformed starts, and blocks
        outside the pool or whose earlier rows are not there (``advance``), are skipped and set
        device error bit 2 (``kernels.device_status``); the rest is written."""

        kernels.block8_write(self, key, value, starts)

    def read(self, rows: int, *, starts: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """The restored last tokens of every sequence, ``rows`` in all, laid
        out as in ``write``: (key, value) [rows, kv_heads, head_dim]."""

        return kernels.block8_read(self, rows, starts)

    def select(self, query: torch.Tensor, *, count: int, first: int = 1, recent: int = 2) -> torch.Tensor:
        """int32 [num_seqs, kv_heads, count]: the ``first`` and the ``recent``
        last blocks and those with the largest bound on the logits of query
        [num_seqs, q_heads, head_dim], ascending, -1 past the end.

        The bound of a block is sum_d max(q_d low_d, q_d high_d) over the
        smallest and largest key of each channel, the query rounded to 8
        bits, its largest value over the KV head's query heads taken: whole-number
        arithmetic and two fp32 products, so equal scores are exactly equal and
        go to the lower block."""

        return kernels.block8_select(query, self, count=count, first=first, recent=recent)

    def attention(self, query: torch.Tensor, *, blocks: torch.Tensor | None = None,
                  softmax_scale: float | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """Causal attention of each sequence's last query tokens, [num_seqs,
        q_heads, head_dim] or [num_seqs, queries, q_heads, head_dim] (up to 16),
        over its tokens, or over those of ``blocks`` (``select``): (out, lse).
        A query that sees no token gives zeros and an LSE of -inf."""

        return kernels.block8_attention(query, self, blocks=blocks, softmax_scale=softmax_scale)

    def attention_workspace(self, queries: int, q_heads: int) -> torch.Tensor:
        """Scratch of one attention launch, on the current stream."""

        size = self._workspace_bytes.get((queries, q_heads))
        if size is None:
            with torch.cuda.device(self.index):  # the multiprocessors of the device that the launch will be on
                size = int(_capi.load().ucb_block8_attention_workspace_bytes(self.descriptor, queries, q_heads))
            if size < 0:
                raise RuntimeError("the device of the block cache is unavailable")
            self._workspace_bytes[(queries, q_heads)] = size
        return self.key_code.new_empty(size)

    def empty(self, dtype: torch.dtype, shape: tuple) -> torch.Tensor:
        """An uninitialised tensor of a launch's output, by the pattern of one expanded element (0.6 us a call less than
        naming type and device)."""

        pattern = self._shapes.get((dtype, shape))
        if pattern is None:
            if len(self._shapes) >= 64:
                self._shapes.clear()
            pattern = self._shapes[(dtype, shape)] = torch.empty(1, device=self.device, dtype=dtype).expand(shape)
        return torch.empty_like(pattern, memory_format=torch.contiguous_format)

    # ---------------------------------------------------------------- accounting
    @property
    def resident_bytes(self) -> int:
        return sum(self.byte_breakdown.values())

    @property
    def byte_breakdown(self) -> dict[str, int]:
        return {
            "payload_bytes": tensor_bytes(self.key_code) + tensor_bytes(self.value_code),
            "scale_bytes": tensor_bytes(self.key_scale) + tensor_bytes(self.value_scale),
            "bound_bytes": tensor_bytes(self.key_low) + tensor_bytes(self.key_high),
            "pending_bytes": tensor_bytes(self.pending_key) + tensor_bytes(self.pending_value),
            "indices_bytes": tensor_bytes(self.block_table) + tensor_bytes(self.lengths),
        }
