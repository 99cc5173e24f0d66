"""The blocks of 8-bit block caches, given to sequences and taken back on the device.

The reference's segments own their memory (unicache/storage/physical.py:204-332);
blocks of a pool can be shared: a prompt continued in several samples is held
once.  Table, lengths and reference counts are device tensors that the calls
here change in stream order without the host, so a step that needs blocks can
be captured as a CUDA graph.
"""

from __future__ import annotations

import ctypes

import torch

from .. import _capi, kernels
from .int8_block import BLOCK_SIZES, Int8BlockCache


class BlockPool:
    """Blocks of one table, for all ``Int8BlockCache`` layers that share it.

    ``block_table`` int32 [num_seqs, max_blocks]: a sequence's blocks, -1 behind them;
    ``lengths`` int32 [num_seqs]; ``references`` int32 [num_blocks]: how many table entries name
    a block, 0 for a free one; ``held`` int32 [num_seqs]: how many blocks a sequence
    has.  Only this object's methods may change table, references and held.  A block that is taken
    is the lowest free one, and sequences are served in ascending order, so the same calls give the same table.

    ``cache`` makes a layer's cache over the pool, ``attach`` takes existing ones: ``fork`` and ``compact`` move
    the contents of all of them.  The methods run on the current stream of the pool's device; like any
    tensors, uses on two streams need an event between them.  What cannot be done sets device error bit 2
    (``kernels.device_status``).
    """

    def __init__(self, *, block_table: torch.Tensor, lengths: torch.Tensor, references: torch.Tensor, block_size: int):
        kernels.require_cuda(block_table, "block_table")
        if block_table.dim() != 2 or references.dim() != 1:
            raise ValueError("block_table must be [num_seqs, max_blocks], references [num_blocks]")
        seqs, width = map(int, block_table.shape)
        if block_size not in BLOCK_SIZES:
            raise ValueError(f"the block pool takes block sizes {BLOCK_SIZES}")
        if not 1 <= seqs <= 4096 or width < 1 or references.numel() < 1:
            raise ValueError("the block pool needs 1 to 4096 sequences and at least one block")
        for name, tensor, shape in (("block_table", block_table, (seqs, width)), ("lengths", lengths, (seqs,)),
                                    ("references", references, tuple(references.shape))):
            if tensor.dtype is not torch.int32 or tuple(tensor.shape) != shape or tensor.device != block_table.device \
                    or not tensor.is_contiguous():
                raise ValueError(f"{name} must be a contiguous int32 tensor of shape {shape} on the pool's device")
        if references.data_ptr() % 16:
            raise ValueError("references must be 16-byte aligned")
        self.block_table, self.lengths, self.references = block_table, lengths, references
        self.held = (block_table >= 0).sum(1, dtype=torch.int32)
        self.device, self.index = block_table.device, block_table.get_device()
        self.num_seqs, self.num_blocks, self.block_size, self.max_tokens = seqs, references.numel(), block_size, width * block_size
        self._struct = _capi.UcbBlockPool(
            block_table=block_table.data_ptr(), lengths=lengths.data_ptr(), held=self.held.data_ptr(),
            references=references.data_ptr(), num_blocks=self.num_blocks, num_seqs=seqs, max_blocks=width,
            block_tokens=block_size)
        self.descriptor = ctypes.addressof(self._struct)
        self.caches: list[Int8BlockCache] = []
        self._layers: list[torch.Tensor] = []  # the caches' descriptors on the device
        self._layers_at, self._kv_heads = None, 0
        self._compact_bytes = int(_capi.load().ucb_block_pool_compact_workspace_bytes(self.descriptor))
        if self._compact_bytes < 0:
            _capi.check(_capi.UCB_ERR_INVALID, "BlockPool")

    @classmethod
    def allocate(cls, num_seqs: int, max_tokens: int, num_blocks: int, *, block_size: int = 64,
                 device: torch.device | str = "cuda") -> "BlockPool":
        """A pool of ``num_blocks`` free blocks for ``num_seqs`` empty sequences of up to ``max_tokens`` tokens."""

        device = torch.device(device)
        if device.type != "cuda":
            raise RuntimeError("the block pool lives on a CUDA device: the b200 backend has no CPU path")
        if device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        if num_seqs < 1 or max_tokens < 1 or num_blocks < 1 or block_size not in BLOCK_SIZES:
            raise ValueError(f"need num_seqs, max_tokens and num_blocks of at least 1 and a block size of {BLOCK_SIZES}")
        table = torch.full((num_seqs, -(-max_tokens // block_size)), -1, device=device, dtype=torch.int32)
        return cls(block_table=table, lengths=torch.zeros(num_seqs, device=device, dtype=torch.int32),
                   references=torch.zeros(num_blocks, device=device, dtype=torch.int32), block_size=block_size)

    def cache(self, *, num_kv_heads: int, head_dim: int = 128, dtype: torch.dtype = torch.bfloat16) -> Int8BlockCache:
        """An empty cache of one layer over this pool, attached to it."""

        cache = Int8BlockCache.allocate(self.num_seqs, self.max_tokens, num_kv_heads=num_kv_heads, head_dim=head_dim,
                                        block_size=self.block_size, dtype=dtype, device=self.device,
                                        block_table=self.block_table, num_blocks=self.num_blocks, lengths=self.lengths)
        self.attach([cache])
        return cache

    def attach(self, caches: list) -> None:
        """Caches whose blocks move with this pool's; they share its table and lengths.  Not while a graph is captured;
        a graph that was captured before goes on with the caches of its time."""

        for cache in caches:
            if cache.block_table.data_ptr() != self.block_table.data_ptr() or cache.lengths.data_ptr() != self.lengths.data_ptr() \
                    or cache.block_table.shape != self.block_table.shape or cache.device != self.device:
                raise ValueError("an attached cache must share the pool's block_table and lengths")
            if int(cache.key_code.shape[0]) != self.num_blocks or cache.block_size != self.block_size:
                raise ValueError("an attached cache must have the pool's blocks and block size")
            if any(cache is other for other in self.caches):
                raise ValueError("the cache is attached already")
        every = [*self.caches, *caches]
        if not every:
            return
        raw = b"".join(ctypes.string_at(c.descriptor, ctypes.sizeof(_capi.UcbBlock8Cache)) for c in every)
        # a new tensor beside the old ones, which graphs that were captured with them still read
        self._layers.append(torch.frombuffer(bytearray(raw), dtype=torch.uint8).to(self.device))
        self._layers_at, self._kv_heads, self.caches = self._layers[-1].data_ptr(), max(c.num_kv_heads for c in every), every

    # ---------------------------------------------------------------- use
    def advance(self, tokens) -> None:
        """Add ``tokens`` (a number or an int32 [num_seqs] tensor) to the lengths before the write of that many rows, and
        give each sequence the blocks that it needs for them.  Takes the place of ``Int8BlockCache.advance``; negative
        numbers withdraw rows as there, and the blocks behind the new end stay the sequence's.

        Where the pool runs out the lengths count all the same, so that writes skip the missing blocks and ``advance`` of
        the negative numbers takes the step back; a length below 0 becomes 0.  A length that would go back into the middle of a block
        that other sequences share stays, as the next write would change their rows (device error bit 2).  It may go back to
        such a block's start, or to nothing: when the sequence grows again it gives the shared blocks back and takes its own."""

        if isinstance(tokens, torch.Tensor):
            at, each = self._indices("tokens", tokens), 0
            if tokens.numel() != self.num_seqs:
                raise ValueError("tokens must have one entry for each sequence")
        else:
            at, each = None, int(tokens)
            if not -(1 << 31) <= each < 1 << 31:
                raise ValueError("tokens must fit 32 bits")
        kernels._call_on(self.index, "ucb_block_pool_advance", self.descriptor, at, each, kernels.stream_of(self.lengths))

    def release(self, sequences: torch.Tensor) -> None:
        """End the sequences (int32 [n]): lengths 0, no blocks.  A block is free once no other sequence shares it."""

        at = self._indices("sequences", sequences)
        kernels._call_on(self.index, "ucb_block_pool_release", self.descriptor, at, sequences.numel(),
                         kernels.stream_of(self.lengths))

    def fork(self, parents: torch.Tensor, children: torch.Tensor) -> None:
        """Sequence ``children[i]`` becomes a copy of ``parents[i]`` (int32 [n] each): what it held is released, the parent's
        complete blocks are shared and its incomplete block is copied in every attached cache.  The rows that the parent's length
        counts are written, and its drafts verified, before: a write into the middle of a block that a fork at its end has shared is
        refused (device error bit 2).

        No sequence may be a child twice, or parent and child in one call: such pairs are skipped.  A beam
        search lets a surviving beam stay where it is and forks only the further ones into
        ended beams.  A child for whose block there is no room is left empty."""

        first, second = self._indices("parents", parents), self._indices("children", children)
        pairs = parents.numel()
        if children.numel() != pairs or pairs > self.num_seqs:
            raise ValueError("parents and children must be of one length, at most num_seqs")
        self._need_caches()
        workspace = self.lengths.new_empty(4 * pairs)
        kernels._call_on(self.index, "ucb_block_pool_fork", self.descriptor, first, second, pairs, self._layers_at,
                         len(self.caches), self._kv_heads, workspace.data_ptr(), kernels.stream_of(self.lengths))

    def compact(self) -> torch.Tensor:
        """Move the blocks in use to the front of the pool in every attached cache: int32 [1], how many they are.

        Of n of them, those at n and behind go to the free blocks in front of n, both in ascending order; the contents of the
        blocks behind are then of no use, so that a pool can be cut or handed on."""

        self._need_caches()
        workspace, live = self.lengths.new_empty(self._compact_bytes // 4), self.lengths.new_empty(1)
        kernels._call_on(self.index, "ucb_block_pool_compact", self.descriptor, self._layers_at, len(self.caches),
                         self._kv_heads, live.data_ptr(), workspace.data_ptr(), kernels.stream_of(self.lengths))
        return live

    def free_blocks(self) -> int:
        """Blocks that no sequence names.  Waits for the device."""

        return int((self.references == 0).sum())

    def _indices(self, name: str, x: torch.Tensor) -> int:
        if not isinstance(x, torch.Tensor) or x.dtype is not torch.int32 or x.get_device() != self.index or x.dim() != 1 \
                or not x.is_contiguous():
            raise ValueError(f"{name} must be a contiguous one-dimensional int32 tensor on the pool's device")
        return x.data_ptr()

    def _need_caches(self) -> None:
        if not self.caches:
            raise ValueError("the block pool has no caches attached: their blocks could not follow")
