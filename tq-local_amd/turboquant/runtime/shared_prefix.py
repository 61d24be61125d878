"""A packed prompt that several sequences continue: one copy of it for all of them.

``share_prefix(cache, sequences)`` turns the packed layers of a prefilled cache [P rows] into layers whose prompt row p
is continued by so many sequences of a batch.  The prompt stays packed once, every sequence has a packed layer of its own
behind it, and a decode step reads the prompt once for all of its sequences
(``turboquant.runtime.shared_prefix_attention``).  ``batch_repeat_interleave`` of a packed layer copies the prompt
instead; layers that the kernel does not take (outlier-split ones, ones kept dense) are copied so.
"""

from __future__ import annotations

from typing import Any, Sequence

import torch
from transformers.cache_utils import Cache, CacheLayerMixin

from turboquant.runtime import kernels as K
from turboquant.runtime.packed_qmse_cache import PackedMSELayer


class SharedPrefixLayer(CacheLayerMixin):
    """One decoder layer's cache for sequences that continue the rows of ``prefix``: row p by ``counts[p]`` of them, those of
    row 0 first."""

    is_sliding = False
    is_compileable = False
    #: what the attention backend knows such a layer by
    shares_prompts = True

    def __init__(self, prefix: PackedMSELayer, counts: Sequence[int]):
        super().__init__()
        store = prefix._store
        if store is None or prefix._split is not None or prefix._dense_len or prefix._force_dense:
            raise ValueError("a shared prefix needs a one-group layer with all of its tokens packed")
        if len(counts) != store.B:
            raise ValueError(f"{len(counts)} numbers of sequences for {store.B} prompts")
        self.prefix = prefix
        self.own = self.without_tokens()
        self.is_initialized = True
        self.device, self.dtype = prefix.device, prefix.dtype
        self._force_dense = False
        self._set_counts([int(n) for n in counts])

    def _set_counts(self, counts: list[int]) -> None:
        self._check_counts(counts)
        self.counts = counts
        dev = self.prefix._store.device
        ends = torch.tensor(counts).cumsum(0)
        #: the prompt of each sequence, and each prompt's first one (any, where it has none)
        self.prompt_of = torch.arange(len(counts)).repeat_interleave(torch.tensor(counts)).to(dev)
        self.first_of = (ends - torch.tensor(counts)).clamp(max=sum(counts) - 1).to(dev)
        even = len(set(counts)) == 1
        self.cu_rows = None if even else torch.cat((torch.zeros(1, dtype=torch.int64), ends)).int().to(dev)

    def without_tokens(self) -> PackedMSELayer:
        """A layer of the prompts' codec that holds nothing."""
        p = self.prefix
        layer = PackedMSELayer(p.bits, p.seed, p.grid_size, use_qjl_keys=p.use_qjl_keys, quantize_decode=p.quantize_decode,
                               reserve_tokens=p.reserve_tokens)
        layer.codecs, layer.device, layer.dtype, layer.is_initialized = p.codecs, p.device, p.dtype, True
        return layer

    @staticmethod
    def _check_counts(counts: list[int]) -> None:
        if min(counts) < 0 or sum(counts) == 0:
            raise ValueError(f"{counts} sequences")

    @property
    def batch(self) -> int:
        return sum(self.counts)

    @property
    def _lazy_update(self) -> bool:
        return self.own._lazy_update

    @_lazy_update.setter
    def _lazy_update(self, on: bool) -> None:
        self.own._lazy_update = on

    # ------------------------------------------------------------ HF protocol
    def lazy_initialization(self, key_states: torch.Tensor, value_states: torch.Tensor) -> None:
        """Nothing is left to do: the prompt came with its codecs."""

    def update(self, key_states: torch.Tensor, value_states: torch.Tensor, *args: Any,
               **kwargs: Any) -> tuple[torch.Tensor, torch.Tensor]:
        """Stores the sequences' new tokens.  With the TurboQuant attention backend wired they are what is returned;
        otherwise every sequence's decoded history with them."""
        if int(key_states.shape[0]) != self.batch:
            raise ValueError(f"{int(key_states.shape[0])} rows for {self.batch} sequences")
        if self.own._lazy_update:
            return self.own.update(key_states, value_states, *args, **kwargs)
        before = self.dense_rows()
        if self.own.quantize_decode:
            self.own._append_packed(key_states, value_states)
        else:
            self.own._append_dense(key_states, value_states)
        return tuple(torch.cat((a, b), dim=2) for a, b in zip(before, (key_states, value_states)))

    def dense_rows(self) -> tuple[torch.Tensor, torch.Tensor]:
        """Every sequence's keys and values [B, H, n, D], decoded: its prompt's, its own packed ones, its dense ones."""
        own = self.own
        keys = [self.prefix._decode_keys_full()[self.prompt_of], own._decode_keys_full(), own._dense_keys]
        values = [self.prefix._decode_values_full()[self.prompt_of], own._decode_values_full(), own._dense_values]
        return tuple(torch.cat([t for t in ts if t is not None and t.shape[2]] or [ts[0]], dim=2) for ts in (keys, values))

    def get_seq_length(self) -> int:
        return self.prefix.packed_seq_length() + self.own.get_seq_length()

    def get_mask_sizes(self, query_length: int) -> tuple[int, int]:
        if torch.is_tensor(query_length):  # older callers pass cache_position
            query_length = int(query_length.shape[0])
        return self.get_seq_length() + int(query_length), 0

    def get_max_length(self) -> int:
        return -1

    def get_max_cache_shape(self) -> int:
        return -1

    def storage_bytes(self) -> int:
        return self.prefix.storage_bytes() + self.own.storage_bytes()

    # ------------------------------------------- rows and tokens chosen and moved
    def _take(self, rows: torch.Tensor) -> None:
        """The sequences ``rows`` (numbers on the host), which stay with their prompts."""
        if rows.numel() and (int(rows.min()) < 0 or int(rows.max()) >= self.batch):
            raise IndexError(f"rows {rows.tolist()} of a batch of {self.batch}")
        prompts = self.prompt_of.cpu()[rows]
        if (prompts.diff() < 0).any():
            raise ValueError(f"rows {rows.tolist()} do not keep the sequences in the order of their prompts")
        counts = torch.bincount(prompts, minlength=len(self.counts)).tolist()
        self._check_counts(counts)
        if self.own._batch() is not None:
            self.own._take_rows(rows)
        self._set_counts(counts)

    def reorder_cache(self, beam_idx: torch.Tensor) -> None:
        """Sequence r becomes sequence beam_idx[r], one of the same prompt (the numbers are looked at on the host)."""
        rows = beam_idx.cpu()
        if rows.shape != (self.batch,) or (rows.numel() and (int(rows.min()) < 0 or int(rows.max()) >= self.batch)):
            raise IndexError(f"rows {rows.tolist()} for a batch of {self.batch}")
        prompts = self.prompt_of.cpu()
        if not torch.equal(prompts[rows], prompts):
            raise ValueError(f"rows {rows.tolist()} take sequences to another prompt")
        if self.own._batch() is not None:
            self.own._take_rows(beam_idx)

    def batch_select_indices(self, indices: torch.Tensor) -> None:
        """Only these sequences (numbers, negative ones from the last, or a bool for each), in the order of their prompts."""
        rows = indices.cpu()
        if rows.dtype == torch.bool:
            if rows.shape != (self.batch,):
                raise IndexError(f"a mask of {tuple(rows.shape)} for a batch of {self.batch}")
            rows = rows.nonzero().flatten()
        self._take(torch.where(rows < 0, rows + self.batch, rows))

    def batch_repeat_interleave(self, repeats: int) -> None:
        """Every sequence ``repeats`` times."""
        if repeats < 1:
            raise ValueError(f"{repeats} repeats")
        self.own.batch_repeat_interleave(repeats)
        self._set_counts([n * repeats for n in self.counts])

    def crop(self, tokens_to_remove: int) -> None:
        """As ``PackedMSELayer.crop``, the sequences' own tokens first."""
        n, total = int(tokens_to_remove), self.get_seq_length()
        drop = min(-n, total) if n < 0 else max(total - n, 0) if n else 0
        mine = min(drop, self.own.get_seq_length())
        if mine:
            self.own.crop(-mine)
        if drop > mine:
            self.prefix.crop(-(drop - mine))

    def keep_tokens(self, index: torch.Tensor, tokens: int | None = None) -> None:
        """As ``PackedMSELayer.keep_tokens``, of the sequences' own tokens."""
        mine = self.own.get_seq_length()
        tokens = mine if tokens is None else int(tokens)
        if tokens > mine:
            raise ValueError(f"keep_tokens: {tokens} tokens, but the last {mine} are the sequences' own")
        self.own.keep_tokens(index, tokens)


def share_prefix(cache: Cache, sequences: int | Sequence[int]) -> Cache:
    """A cache whose prompts are continued by several sequences each: ``sequences`` of them for every row, or a number for each.

    The packed layers of ``cache`` become the shared prompts of the result's layers; they are not copied, and the given cache is to
    be used no further; the attention backend is switched on for the new one.  Layers that cannot be shared are copied for every
    sequence.  Shared layers attend to all of their tokens: a choice of blocks (``attend_blocks``) is refused."""
    per_layer = []  # looked over before any layer is changed
    for layer in cache.layers:
        if not isinstance(layer, PackedMSELayer):
            raise ValueError(f"share_prefix takes packed layers, got {type(layer).__name__}")
        batch = layer._batch()
        if batch is None:
            raise ValueError("share_prefix: the prompts are not in the cache yet")
        if layer._choice is not None:
            raise ValueError("share_prefix: a layer attends to chosen blocks (attend_blocks(None) ends that)")
        counts = [int(sequences)] * batch if isinstance(sequences, int) else [int(n) for n in sequences]
        if len(counts) != batch or min(counts) < 0 or sum(counts) == 0:
            raise ValueError(f"share_prefix: {counts} sequences for {batch} prompts")
        per_layer.append((batch, counts))
    layers = []
    for layer, (batch, counts) in zip(cache.layers, per_layer):
        if layer._store is not None and layer._split is None and not layer._dense_len and layer._store.length \
                and layer._shape[2] == K.HEAD_DIM:
            layers.append(SharedPrefixLayer(layer, counts))
        else:
            layer._take_rows(torch.arange(batch).repeat_interleave(torch.tensor(counts)))
            layers.append(layer)
    return Cache(layers=layers)
