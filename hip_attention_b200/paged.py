"""A page pool of keys and values, next to the sparse attention that reads it: which sequence has which pages
(``HiPPagePool``), new keys and values into their pages (``write_paged_kv``), and exact attention of one new token per
sequence (``paged_decode_attention``) for the layers a server keeps dense.

The pools, tables and lengths are the ones ``hip_attention_12`` takes (``args.k_cache / v_cache / block_table /
cache_seq_lens``) and, with pages of one token, ``forward_paged_hip`` (``req_to_tokens``).  The reference leaves these to the
inference server around it; its configuration has switches for a server that decodes densely (``hip_config.py:97-102``).

The exact attention uses keys as they lie in the pool, so they are rotated before they are written.  With ``using_extend``, the
configuration's default, the sparse attention rotates keys itself and its pools hold them un-rotated: a layer is then exact in all of its
steps, with a pool of rotated keys, or sparse in all of them.  Without ``using_extend`` both read one pool.

Every call is stream-ordered on the current stream of the caches' device, synchronises nothing and can be captured into a
CUDA graph.  They are calls of a server: no gradient passes through them.  What the device finds wrong is recorded in the status word
(``read_status``): HIPATTN_STATUS_NO_PAGES (16), a pool had too few free pages; HIPATTN_STATUS_SEQUENCE (32), a call named a sequence
it cannot take; pages and positions out of range as in the rest of the package.
"""
from __future__ import annotations

from typing import Optional, Sequence, Union

import torch
from torch import Tensor

from .operator import host


def paged_decode_attention(q: Tensor, k_cache: Tensor, v_cache: Tensor, block_table: Tensor, cache_seq_lens: Tensor, *,
                           rows: Optional[Tensor] = None, sm_scale: float = 1.0, sliding_window: Optional[int] = None,
                           logit_softcap: Optional[float] = None, return_lse: bool = False, out: Optional[Tensor] = None):
    """Exact attention of one new token per sequence over its pages.

    ``q`` [B, H, D]; ``k_cache`` / ``v_cache`` [n_pages, page_size, HKV, D] of q's type (float32, float16, bfloat16; D up to
    256) or float8_e5m2 (or its uint8 view) with 16-bit queries; ``block_table`` [R, W] and ``cache_seq_lens`` [R], int32 or
    int64, the lengths counting the new token, whose key and value are in the pool already.  ``rows`` [B]: entry b attends
    sequence rows[b] (None: b; negative: an empty place of a padded batch).  Logits are ``sm_scale`` * q.k (1: q carries the
    scale, as for ``hip_attention_12``), ``logit_softcap`` * tanh(x / logit_softcap) of it when given; with
    ``sliding_window`` only the last so many positions are attended.  Keys are used as they lie in the pool: rotate them
    before they are written.

    How the work is laid out follows from the width of ``block_table``, which is all the host knows of the lengths: give the
    columns that the longest sequence can need (``block_table[:, :w]``; one bfloat16 sequence of 389 tokens, 32 heads over 8 of
    dimension 128, takes 6.7 us behind a table of 448 tokens and 12 us behind one of 131072).

    Returns the context [B, H, D] (in ``out`` when given) and, with ``return_lse``, the base-2 log-sum-exp [B, H] (float32).
    A sequence without tokens gives zeros and -inf."""
    return host().paged_decode(q, k_cache, v_cache, block_table, cache_seq_lens, rows, sm_scale, sliding_window, logit_softcap, return_lse, out)


def write_paged_kv(k: Tensor, v: Tensor, k_cache: Tensor, v_cache: Tensor, block_table: Tensor, cache_seq_lens: Tensor, *,
                   rows: Optional[Tensor] = None, token_offsets: Optional[Tensor] = None) -> None:
    """Writes new keys and values into the pages of their sequences.

    ``k`` / ``v`` [N, HKV, D]: the last tokens of the sequences, whose lengths ``cache_seq_lens`` count them already
    (``HiPPagePool.extend``).  Sequence b (row rows[b] of the table; None: b; negative: its tokens are left out) has tokens
    token_offsets[b] : token_offsets[b + 1], or N / B of them each; tokens outside the offsets are not written.  Give the rows that grew
    (``HiPPagePool.extend``): a growth that was refused has no place for its tokens, and they would go over the last ones.  A
    float8_e5m2 pool (or its uint8 view) receives the nearest values (ties to even, beyond the range infinity).  The rows of a
    call must differ: of two that are the same, which values stay is not defined."""
    host().write_kv(k, v, k_cache, v_cache, block_table, cache_seq_lens, rows, token_offsets)


class HiPPagePool:
    """The pages of the K and V caches of all layers and which sequence reads which of them.

    ``k_caches`` / ``v_caches``: one [n_pages, page_size, HKV, D] tensor per layer, all of one shape, type and layout (the
    tokens of a page contiguous).  Up to ``max_sequences`` sequences (the rows of the table) of up to
    ``max_pages_per_sequence`` pages each.  State, all int32 on the device in one buffer (``state``, so that a checkpoint is one copy):

    * ``ref_counts`` [n_pages]: how many sequences read a page; 0: free;
    * ``seq_lens`` [max_sequences]: tokens of each sequence;
    * ``block_table`` [max_sequences, max_pages_per_sequence]: its pages; entries behind them mean nothing.

    A page that several sequences read is full and is not written again.  Pages are dealt out lowest number first, in the
    order of a call's entries.  An ``extend`` or ``fork`` that cannot be carried out as a whole (too few free pages, a sequence outside
    the table, named twice, not empty or too long) changes nothing and leaves its bit in the status word; ``free`` takes every row
    for itself.  Entries that are negative are left out, so a captured call can be replayed with fewer of them; a call takes up to
    4096.  Calls on one pool, and calls that read its tables, have to be ordered: one stream, or events."""

    def __init__(self, k_caches: Sequence[Tensor], v_caches: Sequence[Tensor], max_sequences: int, max_pages_per_sequence: int) -> None:
        k_caches, v_caches = list(k_caches), list(v_caches)
        if not k_caches or len(k_caches) != len(v_caches):
            raise ValueError(f"one K and one V cache per layer: {len(k_caches)} and {len(v_caches)} were given")
        if not 0 < max_sequences <= 262144 or not 0 < max_pages_per_sequence < 2 ** 31:
            raise ValueError("max_sequences must lie in 1..262144 and max_pages_per_sequence must be positive")
        first = k_caches[0]
        if not isinstance(first, Tensor) or first.ndim != 4:
            raise ValueError("caches must be [n_pages, page_size, kv_heads, head_dim]")
        if not first.is_cuda:
            raise ValueError("the caches must be CUDA tensors: there is no CPU path")
        n_pages, self.page_size = first.shape[:2]
        if n_pages > 0x7fff0000:
            raise ValueError(f"a pool has at most {0x7fff0000} pages, {n_pages} were given")
        self.k_caches, self.v_caches = k_caches, v_caches
        self.state = torch.zeros(n_pages + max_sequences + max_sequences * max_pages_per_sequence, dtype=torch.int32, device=first.device)
        self.ref_counts = self.state[:n_pages]
        self.seq_lens = self.state[n_pages:n_pages + max_sequences]
        self.block_table = self.state[n_pages + max_sequences:].view(max_sequences, max_pages_per_sequence)
        self._handle = host().page_pool(k_caches + v_caches, self.ref_counts, self.seq_lens, self.block_table)

    def extend(self, rows: Tensor, n_tokens: Union[Tensor, int], grown: Optional[Tensor] = None) -> Optional[Tensor]:
        """Sequence rows[i] grows by n_tokens[i] tokens (an int: by as many each) and gets the pages for them.

        ``grown`` (int32, as long as ``rows``) receives the rows that grew, ``rows`` or, when the call could not be carried out, -1
        everywhere, and is returned.  It is what the ``write_paged_kv`` and ``paged_decode_attention`` that follow take as their ``rows``:
        they leave -1 out.  With the rows that were asked for, the tokens of a refused growth would be written over the last ones
        of their sequences, in a page that others may share."""
        return host().pool_extend(self._handle, rows, n_tokens, grown)

    def fork(self, parents: Tensor, children: Tensor) -> None:
        """Sequence children[i], which is empty, becomes a copy of parents[i] (a parent may have several children).  Full
        pages are shared; the tokens of a begun page are copied, in all layers, to a page of the child's own."""
        host().pool_fork(self._handle, parents, children)

    def free(self, rows: Tensor) -> None:
        """The sequences become empty; pages that no other sequence reads are free again.  Naming a row twice frees it once; a
        row beyond the table leaves its bit in the status word, the others are freed."""
        host().pool_free(self._handle, rows)

    def compact(self) -> Tensor:
        """Moves the pages in use to the front of the pool, in all layers, and renames them in the tables: with m pages in
        use, those numbered m and more go, ascending, to the free ones below m.  Returns m (int32 [1], on the device)."""
        return host().pool_compact(self._handle)
