"""paged.py -- PagedErrorCorrectedCache: the compressed cache in pages, for
sequences of different lengths (no counterpart in the reference, whose cache
holds one contiguous row per sequence and one length for the batch).

Per layer a K and a V pool of 128-byte blocks (or 96-byte records), ``[pages,
Hkv, page_size, block_bytes]``; one page table ``[slots, max_cache_len /
page_size]`` for all layers; lengths in device memory.  Pages are taken as
sequences grow and given back by ``release`` and ``evict``.  Appends, decode
attention and eviction are the paged operators of ``custom_ecc_cuda``.
"""
from __future__ import annotations

from typing import Any, Dict, List, Optional, Sequence, Tuple

import torch

import custom_ecc_cuda as ops

from .cache import BLOCK_BYTES, HEAD_DIM, RECORD96, _HFCache


class PagedErrorCorrectedCache(_HFCache):
    """HF cache of ``batch_size`` slots whose sequences grow and end on their
    own.  Pass as ``past_key_values`` with the SDPA patch active
    (``paged_ecc_cache`` or ``patch_model``), or call ``append`` and
    ``decode_attention`` directly.

    ``num_pages``: pages per layer (default: enough for every slot at
    ``max_cache_len``).  ``window`` / ``sinks``: decode attends to the last
    ``window`` tokens and the first ``sinks`` only.  ``collect_weights``: decode
    adds up the attention weight of every cached token, by which ``evict`` cuts
    the sequences to a budget.

    Sequences hold no padding: a batch is appended at the end of every slot's
    own sequence, and an attention mask that hides cached tokens is refused.
    A model takes one position for all slots unless it is told otherwise: with
    slots of different lengths pass ``position_ids=cache.position_ids()``.
    ``get_seq_length`` counts the tokens seen (positions go on after an
    eviction); ``lengths`` are the tokens held."""

    def __init__(self, config, batch_size: int = 1, max_cache_len: int = 32768, num_pages: Optional[int] = None,
                 page_size: int = 64, device: Optional[str] = None, rotate_values: bool = True, window: int = 0,
                 sinks: int = 0, collect_weights: bool = False, block_bytes: int = BLOCK_BYTES):
        try:
            super().__init__()
        except (TypeError, ValueError):
            pass
        self.layers = []
        dev = torch.device(device) if device is not None else torch.device("cuda")
        if dev.type != "cuda" or not torch.cuda.is_available():
            raise RuntimeError("PagedErrorCorrectedCache needs a CUDA device: the compressed cache lives in GPU memory "
                               "and is read by the sm_100a kernels (there is no CPU path)")
        if dev.index is None:
            dev = torch.device("cuda", torch.cuda.current_device())
        self._device = dev
        self.config = config
        self.batch_size = int(batch_size)
        self.num_heads = getattr(config, "num_key_value_heads", None) or config.num_attention_heads
        self.num_attention_heads = config.num_attention_heads
        self.head_dim = getattr(config, "head_dim", None) or config.hidden_size // config.num_attention_heads
        self._num_layers = int(config.num_hidden_layers)
        self.page_size = int(page_size)
        if self.head_dim != HEAD_DIM:
            raise RuntimeError(f"PagedErrorCorrectedCache stores 128-dim heads; got head_dim={self.head_dim}")
        if self.num_attention_heads % self.num_heads or self.num_attention_heads // self.num_heads > 8:
            raise RuntimeError("the paged decode takes 1 to 8 query heads per kv head")
        if block_bytes not in (BLOCK_BYTES, RECORD96):
            raise RuntimeError(f"block_bytes must be {BLOCK_BYTES} or {RECORD96}, got {block_bytes}")
        if self.page_size < 16 or self.page_size % 16:
            raise RuntimeError(f"page_size must be a multiple of 16, got {page_size}")
        if window < 0 or sinks < 0 or (sinks and not window):
            raise RuntimeError("window and sinks must not be negative, and sinks need a window")
        self.block_bytes, self.rotate_values = int(block_bytes), bool(rotate_values)
        self.window, self.sinks = int(window), int(sinks)
        self._width = -(-int(max_cache_len) // self.page_size)
        self._max_cache_len = self._width * self.page_size
        total = self.batch_size * self._width if num_pages is None else int(num_pages)
        if total < 1:
            raise RuntimeError("num_pages must be positive")
        shape = (self._num_layers, total, self.num_heads, self.page_size, self.block_bytes)
        self._k_pool = torch.zeros(shape, dtype=torch.uint8, device=dev)
        self._v_pool = torch.zeros(shape, dtype=torch.uint8, device=dev)
        self.weights = torch.zeros((self._num_layers, self.batch_size, self.num_heads, self._max_cache_len),
                                   dtype=torch.float32, device=dev) if collect_weights else None
        # host bookkeeping and its device copies
        self._free: List[int] = list(range(total - 1, -1, -1))
        self._pages: List[List[int]] = [[] for _ in range(self.batch_size)]
        self._len: List[int] = [0] * self.batch_size
        self._seen: List[int] = [0] * self.batch_size
        self.block_table = torch.full((self.batch_size, self._width), -1, dtype=torch.int32, device=dev)
        self.seq_lens = torch.zeros(self.batch_size, dtype=torch.int32, device=dev)
        self._pos = torch.zeros(self.batch_size, dtype=torch.int32, device=dev)
        # what patch.py asks to find the layer of a decode call
        self._last_layer = 0
        self._layer_fill: List[int] = [0] * self._num_layers
        self._old_len: List[int] = [0] * self.batch_size
        self._new: Optional[torch.Tensor] = None

    # ------------------------------------------------------------------ #
    # pages                                                               #
    # ------------------------------------------------------------------ #
    @property
    def lengths(self) -> List[int]:
        """Tokens held per slot."""
        return list(self._len)

    def position_ids(self) -> torch.Tensor:
        """The position of every slot's next token, [B, 1] int64 on the GPU."""
        return torch.tensor(self._seen, dtype=torch.int64).to(self._device)[:, None]

    def check_positions(self, position_ids: Optional[torch.Tensor], position_embeddings=None) -> None:
        """Refuses a model's step that rotates slots of different lengths all at one
        position (what a model does by itself: the longest slot's).  Called
        before the first layer with what its attention module is given; with
        slots of different lengths it waits for the GPU."""
        if min(self._seen) == max(self._seen):
            return
        if position_ids is not None:  # [.., B or 1, L]
            per_slot = position_ids.dim() > 1 and position_ids.shape[-2] == self.batch_size
            one = not per_slot or bool((position_ids[..., -1] == max(self._seen)).all())
        elif position_embeddings is not None:  # (cos, sin), [B or 1, L, ..]
            last = position_embeddings[1][:, -1]
            one = last.shape[0] != self.batch_size or bool((last == last[:1]).all())
        else:
            return  # a model that does not show its positions
        if one:
            raise RuntimeError("the slots have different lengths, and the step's positions are the same for all of them: pass "
                               "position_ids=cache.position_ids()")

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def layer_pools(self, layer_idx: int) -> Tuple[torch.Tensor, torch.Tensor]:
        """(K pool, V pool) of one layer, [pages, Hkv, page_size, block_bytes] u8."""
        return self._k_pool[layer_idx], self._v_pool[layer_idx]

    def _upload(self, slots: Sequence[int]) -> None:
        """Device copies of the lengths and of the slots' rows of the table."""
        if slots:
            rows = [self._pages[b] + [-1] * (self._width - len(self._pages[b])) for b in slots]
            at = torch.tensor(list(slots), device=self._device)
            self.block_table[at] = torch.tensor(rows, dtype=torch.int32).to(self._device)
        self.seq_lens.copy_(torch.tensor(self._len, dtype=torch.int32))

    def _grow(self, new: Sequence[int]) -> None:
        """Room for new[b] more tokens in every slot; positions and lengths move on."""
        want = [n + m for n, m in zip(self._len, new)]
        if max(want) > self._max_cache_len:
            raise RuntimeError(f"cache overflow: {max(want)} tokens > max_cache_len {self._max_cache_len}")
        need = [-(-n // self.page_size) - len(p) for n, p in zip(want, self._pages)]
        if sum(need) > len(self._free):
            raise RuntimeError(f"out of pages: {sum(need)} needed, {len(self._free)} free (release or evict sequences)")
        for b, n in enumerate(need):
            self._pages[b] += [self._free.pop() for _ in range(n)]
        self._pos.copy_(self.seq_lens)
        self._old_len = list(self._len)
        self._len = want
        self._seen = [n + m for n, m in zip(self._seen, new)]
        self._upload([b for b, n in enumerate(need) if n])

    def _ungrow(self, before: Tuple[List[int], List[int], List[int], List[int]]) -> None:
        """Takes back a _grow whose tokens were not written; before: (lengths, tokens seen, pages held, lengths before
        the last step) as they were."""
        held = before[2]
        back = [b for b, p in enumerate(self._pages) if len(p) > held[b]]
        for b in reversed(back):
            self._free += reversed(self._pages[b][held[b]:])
            del self._pages[b][held[b]:]
        self._len, self._seen, self._old_len = before[0], before[1], before[3]
        self._upload(back)
        self._pos.copy_(torch.tensor(self._old_len, dtype=torch.int32))

    def release(self, slots: Optional[Sequence[int]] = None) -> None:
        """Ends the sequences of the slots (default: all) and frees their pages."""
        slots = range(self.batch_size) if slots is None else slots
        for b in slots:
            self._free += reversed(self._pages[b])
            self._pages[b], self._len[b], self._seen[b] = [], 0, 0
            if self.weights is not None:
                self.weights[:, b].zero_()
        self._upload(list(slots))
        self._layer_fill = [max(self._seen)] * self._num_layers

    reset = release

    # ------------------------------------------------------------------ #
    # operators                                                           #
    # ------------------------------------------------------------------ #
    def append(self, key_states: torch.Tensor, value_states: torch.Tensor, layer_idx: int,
               new_lens: Optional[Sequence[int]] = None) -> None:
        """Compress the new K/V [B, Hkv, L, 128] of one layer behind every
        slot's sequence; with ``new_lens`` the first new_lens[b] tokens of each
        (the rest is padding).  Layer 0 comes first: it takes the pages and
        moves the lengths, the other layers of the same step follow it."""
        B, H, L, d = key_states.shape
        if d != HEAD_DIM or H != self.num_heads or B != self.batch_size:
            raise RuntimeError(f"append: expected [B={self.batch_size}, H={self.num_heads}, L, 128], "
                               f"got {tuple(key_states.shape)}")
        if value_states.shape != key_states.shape:
            raise RuntimeError(f"append: keys {tuple(key_states.shape)} and values {tuple(value_states.shape)} differ")
        new = [L] * B if new_lens is None else [int(n) for n in new_lens]
        if len(new) != B or min(new) < 0 or max(new) > L:
            raise RuntimeError(f"new_lens must hold {B} counts from 0 to {L}")
        k16 = key_states if key_states.dtype == torch.float16 else key_states.to(torch.float16)
        v16 = value_states if value_states.dtype == torch.float16 else value_states.to(torch.float16)
        if layer_idx == 0:
            before = (self._len, self._seen, [len(p) for p in self._pages], self._old_len)
            last_new = self._new
            self._grow(new)
            try:
                self._new = None if new_lens is None else torch.tensor(new, dtype=torch.int32).to(self._device)
                self._write(k16, v16, 0)
            except Exception:  # refused states, say: the sequences stay as they were
                self._new = last_new
                self._ungrow(before)
                raise
        elif [n + m for n, m in zip(self._old_len, new)] != self._len:
            raise RuntimeError("every layer of a step must append what layer 0 appended")
        else:
            self._write(k16, v16, layer_idx)
        self._last_layer = layer_idx
        self._layer_fill[layer_idx] = max(self._seen)

    def _write(self, k16: torch.Tensor, v16: torch.Tensor, layer_idx: int) -> None:
        kp, vp = self.layer_pools(layer_idx)
        if self.rotate_values:
            ops.compress_pair_paged(k16, v16, kp, vp, self.block_table, self._pos, new_lens=self._new)
        else:
            ops.compress_pair_paged(k16, None, kp, None, self.block_table, self._pos, new_lens=self._new)
            ops.compress_pair_paged(v16, None, vp, None, self.block_table, self._pos, new_lens=self._new, rotate=False)

    def context(self, layer_idx: int) -> Tuple[torch.Tensor, torch.Tensor]:
        """The layer's K and V read back in the model's basis, [B, Hkv, longest
        length, 128] fp16, zeros behind each sequence."""
        kp, vp = self.layer_pools(layer_idx)
        n = max(self._len)
        if self.rotate_values:
            return ops.dequantize_paged(kp, vp, self.block_table, self.seq_lens, n)
        return (ops.dequantize_paged(kp, None, self.block_table, self.seq_lens, n),
                ops.dequantize_paged(vp, None, self.block_table, self.seq_lens, n, unrotate=False))

    def decode_attention(self, query: torch.Tensor, layer_idx: int, sm_scale: Optional[float] = None,
                         attn_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
        """One decode step of attention of ``query`` [B, Hq, 1, 128] over every
        slot's own sequence (the new token already appended).  ``attn_mask`` may
        hide nothing and add nothing (every layer's is looked at, which waits for
        the GPU): sequences hold no padding, and the kernel adds no bias."""
        if attn_mask is not None:
            see = attn_mask if attn_mask.dtype == torch.bool else attn_mask == 0
            if not bool(see.all()):
                raise RuntimeError("PagedErrorCorrectedCache holds no padding and adds no bias: the attention mask hides cached "
                                   "tokens or adds to their scores")
        kp, vp = self.layer_pools(layer_idx)
        q16 = query if query.dtype == torch.float16 else query.to(torch.float16)
        out = ops.decode_attention_paged(q16, kp, vp, self.block_table, self.seq_lens, sm_scale=sm_scale,
                                         window=self.window, sinks=self.sinks, rotate_q=True,
                                         unrotate_out=self.rotate_values,
                                         weights=None if self.weights is None else self.weights[layer_idx])
        return out if query.dtype == torch.float16 else out.to(query.dtype)

    def evict(self, budget: int, sinks: int = 0, recent: int = 0) -> List[int]:
        """Cuts every sequence longer than ``budget`` down to it, in every layer
        and kv head by that head's accumulated weights: the first ``sinks``, the
        last ``recent`` and the heaviest of the others stay, in their order.
        Needs ``collect_weights`` and, per sequence, free pages for the budget;
        the pages held before are free afterwards.  Returns the slots cut."""
        if self.weights is None:
            raise RuntimeError("evict needs collect_weights=True")
        slots = [b for b, n in enumerate(self._len) if n > budget]
        if not slots:
            return slots
        if budget < 1 or sinks < 0 or recent < 0 or sinks + recent > budget:
            raise RuntimeError("budget must be positive and hold the sinks and the recent tokens")
        per = -(-budget // self.page_size)
        if per > len(self._free):
            raise RuntimeError(f"out of pages: an eviction to {budget} tokens needs {per} free, {len(self._free)} are")
        at_once = len(self._free) // per  # sequences whose new pages are free at the same time
        for i in range(0, len(slots), at_once):
            part = slots[i:i + at_once]
            fresh = [[self._free.pop() for _ in range(per)] for _ in part]
            try:
                rows = torch.tensor(part, device=self._device)
                table, lens = self.block_table[rows], self.seq_lens[rows]
                out_table = torch.tensor(fresh, dtype=torch.int32).to(self._device)
                weights = []  # of the kept tokens: they count once every layer is cut
                for layer in range(self._num_layers):
                    kp, vp = self.layer_pools(layer)
                    w, _ = ops.evict_paged(kp, vp, table, lens, self.weights[layer][rows], out_table, budget, sinks=sinks,
                                           recent=recent)
                    weights.append(w[:, :, :budget].clone())
                    del w
            except Exception:  # out of memory, say: the blocks were copied, nothing of the cache has changed
                self._free += [p for pages in reversed(fresh) for p in reversed(pages)]
                raise
            for layer, w in enumerate(weights):
                self.weights[layer, rows, :, :budget] = w
                self.weights[layer, rows, :, budget:] = 0
            for b, pages in zip(part, fresh):
                self._free += reversed(self._pages[b])
                self._pages[b], self._len[b] = pages, budget
            self._upload(part)
        return slots

    # ------------------------------------------------------------------ #
    # HuggingFace Cache protocol                                          #
    # ------------------------------------------------------------------ #
    def update(self, key_states: torch.Tensor, value_states: torch.Tensor, layer_idx: int,
               cache_kwargs: Optional[Dict[str, Any]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """Append and return the K/V attention should use: the new states when
        they are the whole context or a single token (the patched SDPA then
        reads the pages), otherwise the context read back, with the new states
        in the place of their reconstruction (all slots at one length,
        nothing evicted: the model's causal mask counts the tokens seen).  The
        states come rotated: slots of different lengths each at its own position."""
        L = key_states.shape[2]
        if L > 1 and layer_idx == 0 and (min(self._len) != max(self._len) or self._seen != self._len):
            raise RuntimeError("a chunk of several tokens needs all slots at one length and nothing evicted (append and "
                               "attend per sequence)")
        self.append(key_states, value_states, layer_idx)
        if L == 1 or max(self._old_len) == 0:
            return key_states, value_states
        k, v = self.context(layer_idx)
        old = self._old_len[0]
        return (torch.cat([k[:, :, :old].to(key_states.dtype), key_states], dim=-2),
                torch.cat([v[:, :, :old].to(value_states.dtype), value_states], dim=-2))

    def get_seq_length(self, layer_idx: int = 0) -> int:
        return self._layer_fill[layer_idx]

    def get_max_cache_shape(self, layer_idx: int = 0) -> int:
        return self._max_cache_len

    def get_mask_sizes(self, query_length, layer_idx: int = 0) -> tuple:
        if isinstance(query_length, torch.Tensor):
            query_length = int(query_length.shape[0]) if query_length.dim() > 0 else int(query_length)
        return (self.get_seq_length(layer_idx) + int(query_length), 0)

    # What transformers' Cache does to its own layers, which this cache has none of: beams, candidates that are taken
    # back and batches that change are refused, not passed over.
    def crop(self, max_length: int) -> None:
        raise RuntimeError("PagedErrorCorrectedCache cannot be cropped (release() ends a sequence, evict() cuts it)")

    def reorder_cache(self, beam_idx: torch.Tensor) -> None:
        raise RuntimeError("PagedErrorCorrectedCache cannot be reordered: no beam search")

    def batch_repeat_interleave(self, repeats: int) -> None:
        raise RuntimeError("PagedErrorCorrectedCache has a fixed number of slots")

    def batch_select_indices(self, indices: torch.Tensor) -> None:
        raise RuntimeError("PagedErrorCorrectedCache has a fixed number of slots (release() ends a sequence)")

    @property
    def is_compileable(self) -> bool:
        return False

    @property
    def is_initialized(self) -> bool:
        return True

    @property
    def is_sliding(self) -> List[bool]:
        return [False] * self._num_layers

    @property
    def max_batch_size(self) -> int:
        return self.batch_size

    @property
    def max_cache_len(self) -> int:
        return self._max_cache_len

    def __len__(self) -> int:
        return self._num_layers

    def __repr__(self) -> str:
        return (f"PagedErrorCorrectedCache(lengths={self._len}, pages={self._k_pool.shape[1] - len(self._free)}/"
                f"{self._k_pool.shape[1]} of {self.page_size}, layers={self._num_layers})")
