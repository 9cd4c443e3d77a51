"""The attention block's paged cache: its pages, and the attention that reads it.

A cache row is what one token leaves behind for later ones: ``dim`` 16-bit
values that serve every head as key and value (as ``attention.sparse_attn``
takes them).  Rows live in pages, ``pages [(layers,) n_pages, page_size, dim]``;
int32 tables on the device say which pages a sequence holds:

* ``page_table [n_seqs, max_pages]``: a sequence's pages in order, -1 behind the last
* ``seq_lens [n_seqs]``: tokens a sequence has room for
* ``page_refs [n_pages]``: sequences that hold a page; 0 = free

Every function is one call into libdsv4moe.so on torch's current stream and
changes the tables in stream order without reading anything back, so a decode
step (reserve, append, attend) can be captured into a CUDA graph.  Entries that
make no sense (ids out of range, no page at a position, too few free pages) are
skipped and latch a device-side error, read by ``_lib.raise_on_device_error()``.
None of them has a gradient: tensors that require one are refused, except under
``torch.no_grad()`` or in inference mode.

``PagedKVCache`` holds the tensors and calls the functions.
"""

from __future__ import annotations

import torch

from . import ops


def append(pages: torch.Tensor, rows: torch.Tensor, page_table: torch.Tensor, seq_ids: torch.Tensor | None,
           positions: torch.Tensor, freqs: torch.Tensor | None = None, *, interleaved: bool = True,
           offset: int | None = None, amplitude: float = 1.0) -> None:
    """Write rows [T, dim] to positions [T] of the sequences seq_ids [T] (None:
    row t is sequence t's), rotated as ``rotary.rotary`` does when ``freqs`` are
    given.  A negative sequence or position marks padding.  No two rows may name
    the same place."""
    ops.load().cache_append(pages, rows, page_table, seq_ids, positions, freqs, interleaved, offset, float(amplitude))


def paged_attn(q: torch.Tensor, pages: torch.Tensor, page_table: torch.Tensor, seq_ids: torch.Tensor | None,
               positions: torch.Tensor, attn_sink: torch.Tensor | None, softmax_scale: float, *, window: int = 0,
               first: int = 0) -> torch.Tensor:
    """q [T, heads, dim], row t at positions[t] of sequence seq_ids[t] (None: t):
    attention over the sequence's rows 0 .. positions[t], with ``window`` > 0 only
    over the last ``window`` of them and the first ``first`` ones;
    ``attn_sink [heads]`` logits join the denominator.  Several rows may stand in
    one sequence (drafted tokens, a piece of a prompt).  A row with a negative
    sequence or position gives zeros.  1 to 128 heads, dim 128, 256 or 512,
    page_size a power of two from 16 on."""
    return ops.load().paged_attn(q, pages, page_table, seq_ids, positions, attn_sink, float(softmax_scale),
                                 window, first)


def reserve(page_table: torch.Tensor, seq_lens: torch.Tensor, page_refs: torch.Tensor, seqs: torch.Tensor,
            lens: torch.Tensor, page_size: int) -> None:
    """Room for lens[i] tokens in sequence seqs[i]: free pages, lowest id first, in
    the order of the entries; if there are too few, nothing changes.  Negative
    sequences are padding; a sequence may be named once."""
    ops.load().cache_reserve(page_table, seq_lens, page_refs, seqs, lens, page_size)


def free(page_table: torch.Tensor, seq_lens: torch.Tensor, page_refs: torch.Tensor, seqs: torch.Tensor) -> None:
    """The sequences let go of their pages."""
    ops.load().cache_free(page_table, seq_lens, page_refs, seqs)


def fork(pages: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor, page_refs: torch.Tensor,
         parents: torch.Tensor, children: torch.Tensor, lens: torch.Tensor | None = None) -> None:
    """The empty sequence children[i] becomes the first lens[i] tokens (None: all)
    of parents[i].  Full pages are shared; a part-filled last page is copied to a
    free page in every layer, so both may go on writing behind the fork (not before
    it: those pages are the other's too)."""
    ops.load().cache_fork(pages, page_table, seq_lens, page_refs, parents, children, lens)


def compact(pages: torch.Tensor, page_table: torch.Tensor, page_refs: torch.Tensor) -> torch.Tensor:
    """Move the used pages to the lowest ids, in every layer; tables and holder
    counts follow.  Returns int32 [n_pages]: each old id's new one, -1 if free."""
    return ops.load().cache_compact(pages, page_table, page_refs)


def copy_pages(pages: torch.Tensor, src: torch.Tensor, dst: torch.Tensor) -> None:
    """Page src[i] to page dst[i] in every layer.  Negative ids are padding; no
    target may be another entry's source or target."""
    ops.load().cache_copy(pages, src, dst)


class PagedKVCache:
    """``n_pages`` pages of ``page_size`` rows in every one of ``n_layers`` layers,
    shared by ``n_seqs`` sequences of up to ``max_len`` tokens."""

    def __init__(self, n_layers: int, n_pages: int, n_seqs: int, max_len: int, *, page_size: int = 64, dim: int = 512,
                 dtype: torch.dtype = torch.bfloat16, device=None):
        device = torch.device(device) if device is not None else torch.device("cuda")
        self.page_size, self.max_len = page_size, max_len
        max_pages = (max_len + page_size - 1) // page_size
        self.pages = torch.zeros(n_layers, n_pages, page_size, dim, dtype=dtype, device=device)
        self.page_table = torch.full((n_seqs, max_pages), -1, dtype=torch.int32, device=device)
        self.seq_lens = torch.zeros(n_seqs, dtype=torch.int32, device=device)
        self.page_refs = torch.zeros(n_pages, dtype=torch.int32, device=device)

    def reserve(self, seqs: torch.Tensor, lens: torch.Tensor) -> None:
        reserve(self.page_table, self.seq_lens, self.page_refs, seqs, lens, self.page_size)

    def free(self, seqs: torch.Tensor) -> None:
        free(self.page_table, self.seq_lens, self.page_refs, seqs)

    def fork(self, parents: torch.Tensor, children: torch.Tensor, lens: torch.Tensor | None = None) -> None:
        fork(self.pages, self.page_table, self.seq_lens, self.page_refs, parents, children, lens)

    def compact(self) -> torch.Tensor:
        return compact(self.pages, self.page_table, self.page_refs)

    def copy_pages(self, src: torch.Tensor, dst: torch.Tensor) -> None:
        copy_pages(self.pages, src, dst)

    def append(self, layer: int, rows: torch.Tensor, seq_ids: torch.Tensor | None, positions: torch.Tensor,
               freqs: torch.Tensor | None = None, **how) -> None:
        append(self.pages[layer], rows, self.page_table, seq_ids, positions, freqs, **how)

    def attend(self, layer: int, q: torch.Tensor, seq_ids: torch.Tensor | None, positions: torch.Tensor,
               attn_sink: torch.Tensor | None, softmax_scale: float, **mask) -> torch.Tensor:
        return paged_attn(q, self.pages[layer], self.page_table, seq_ids, positions, attn_sink, softmax_scale, **mask)
