"""Pages of the cache as sequences come, branch and go, on the device.

The reference keeps this state on the host (a reference count per page and a
block table per sequence, src/engine/memory/allocator.py); these calls work on
it as int32 device tensors, without a host loop or a synchronisation, so a
step that reorders beams or gives pages back can be captured in a CUDA graph:

* ``ref_counts`` [pages]: holders of a page (tables, a prefix cache); 0 = free
* ``block_tables`` [sequences, max_blocks]: page of tokens [16 j, 16 j + 16)
  of a sequence, -1 where it was given back
* ``seq_lens`` [sequences]: tokens a sequence holds; its pages are the first
  ceil(seq_len / 16) entries, and what lies behind them is not read. Between a
  fork and the append of its token the page of that token is held too: a call
  there counts it, as far as the table has room (``held = (seq_lens + 1).clamp(
  max=16 * max_blocks)``, then ``free_sequences(tables, held, refs)`` or
  ``compact_pages(pool, tables, held, refs)``). A length past the table is an
  error: ``free_sequences`` and ``evict_window_pages`` leave such a row as it
  is, ``compact_pages`` updates the entries that there are.

Each call returns ``counts``, an int32 device tensor of three; its last entry
counts what could not be done (it stays 0 in a sound step), which is also
recorded in the device status (``PA_CHECK=1`` raises it).
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib
from .flashinfer_api import _after, _device_guard, _stream


def _on_gpu_i32(t: torch.Tensor, name: str, dim: int) -> torch.Tensor:
    if t.dtype != torch.int32:
        raise TypeError(f"{name} must be int32")
    if not t.is_cuda:
        raise ValueError(f"{name} must be on the GPU")
    if t.dim() != dim or (t.shape[-1] > 1 and t.stride()[-1] != 1):
        raise ValueError(f"{name} must be {dim}-D with contiguous entries")
    return t


def _state(block_tables, seq_lens, ref_counts) -> torch.device:
    """Checks the three tensors; returns their device."""
    _on_gpu_i32(block_tables, "block_tables", 2)
    _on_gpu_i32(seq_lens, "seq_lens", 1)
    _on_gpu_i32(ref_counts, "ref_counts", 1)
    if seq_lens.numel() != block_tables.size(0):
        raise ValueError("seq_lens must hold one length per row of block_tables")
    if ref_counts.numel() == 0:
        raise ValueError("ref_counts must hold one count per page")
    if not block_tables.device == seq_lens.device == ref_counts.device:
        raise ValueError("block_tables, seq_lens and ref_counts must be on one GPU")
    return block_tables.device


def _row_stride(t: torch.Tensor) -> int:
    """Elements between rows; rows of their own (a broadcast table has one)."""
    rows, width = t.shape
    stride = t.stride()[0]
    if stride >= width:
        return stride
    if rows > 1:
        raise ValueError("the rows of block_tables must not overlap")
    return width


def _page_size(kv_pool: torch.Tensor, kv_layout: str) -> int:
    if kv_layout not in ("HND", "NHD"):
        raise ValueError(f"kv_layout must be 'HND' or 'NHD', not {kv_layout!r}")
    return kv_pool.size(-2 if kv_layout == "HND" else -3)


def _pool(kv_pool: torch.Tensor, ref_counts: torch.Tensor):
    """(pointer, layer stride, layers, page stride, page bytes, pages) in bytes
    of the engine's pool [L, N, 2, H_kv, P, D] or one layer of it."""
    pool = kv_pool if kv_pool.dim() == 6 else kv_pool.unsqueeze(0)
    if pool.dim() != 6 or not pool.is_cuda:
        raise ValueError("kv_pool must be [L, N, 2, H_kv, P, D], for NHD [L, N, 2, P, H_kv, D] "
                         "(or one layer), on the GPU")
    if pool.device != ref_counts.device:
        raise ValueError("kv_pool and ref_counts must be on one GPU")
    if pool.size(1) != ref_counts.numel():
        raise ValueError("ref_counts must hold one count per page of kv_pool")
    size, stride, es = pool.shape, pool.stride(), pool.element_size()
    page = size[2] * size[3] * size[4] * size[5]
    if not pool.is_contiguous():
        at = 1
        for i in (5, 4, 3, 2):  # a page of a layer is one contiguous block
            if size[i] > 1 and stride[i] != at:
                raise ValueError("each page of a layer must be one contiguous block")
            at *= size[i]
        if (size[1] > 1 and stride[1] < page) or (size[0] > 1 and stride[0] < page):
            raise ValueError("the pages of kv_pool must not overlap")
    return (pool.data_ptr(), stride[0] * es, size[0], max(stride[1], page) * es, page * es,
            size[1])


def _release(what, block_tables, seq_lens, ref_counts, page_size, window_left, sinks):
    device = _state(block_tables, seq_lens, ref_counts)
    counts = ref_counts.new_empty(3)
    with _device_guard(device):
        _lib.check(_lib.load().pa_release_pages(
            block_tables.data_ptr(), _row_stride(block_tables), block_tables.shape[1],
            seq_lens.data_ptr(), seq_lens.numel(), int(page_size), window_left, sinks,
            ref_counts.data_ptr(), ref_counts.numel(), counts.data_ptr(), _stream()), what)
        _after(what)
    return counts


def evict_window_pages(block_tables: torch.Tensor, seq_lens: torch.Tensor,
                       ref_counts: torch.Tensor, window_left: int, num_sink_tokens: int = 0,
                       page_size: int = 16) -> torch.Tensor:
    """Gives back the pages that lie wholly behind each sequence's window: with
    ``start = seq_len - 1 - window_left`` the entries from
    ``ceil(num_sink_tokens / page_size)`` up to ``start // page_size`` lose
    their reference and become -1, in place. The sliding-window wrappers with
    this window do not read them, for the last cached token's query and every
    later one. counts: entries given back, pages that became free, errors."""
    window_left, num_sink_tokens = int(window_left), int(num_sink_tokens)
    if not (0 <= window_left < 2 ** 31 and 0 <= num_sink_tokens < 2 ** 31):
        raise ValueError("window_left and num_sink_tokens must be in [0, 2**31)")
    return _release("evict_window_pages", block_tables, seq_lens, ref_counts, page_size,
                    window_left, num_sink_tokens)


def free_sequences(block_tables: torch.Tensor, seq_lens: torch.Tensor, ref_counts: torch.Tensor,
                   page_size: int = 16) -> torch.Tensor:
    """Ends the sequences of these rows: every page loses their reference, the
    entries become -1 and the lengths 0, in place (pass the rows that end, for
    example ``block_tables[3:5], seq_lens[3:5]``). counts as for
    :func:`evict_window_pages`."""
    return _release("free_sequences", block_tables, seq_lens, ref_counts, page_size, -1, 0)


def fork_sequences(kv_pool: torch.Tensor, block_tables: torch.Tensor, seq_lens: torch.Tensor,
                   parents: torch.Tensor, ref_counts: torch.Tensor,
                   out: Optional[torch.Tensor] = None, kv_layout: str = "HND",
                   all_held: bool = False) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Sequence r continues sequence ``parents[r]``: beam search's reordering
    of states, or several samples of one prompt. Returns (block_tables,
    seq_lens, counts) of the new sequences; ``ref_counts`` and ``kv_pool`` are
    updated in place.

    Full pages are shared. The page that the next token goes to is the
    sequence's own: a free page where the length is a multiple of the page
    size, otherwise the parent's unfinished page, kept by the first sequence
    that continues it if nobody else holds it and copied (all layers) into a
    free page for the others. Sequences that nobody continues give up their
    pages; ``parents[r] = -1`` ends sequence r (length 0, entries -1, no page).
    Free pages are those with count 0, taken lowest number first.
    counts: pages copied, pages taken, sequences left without a page (their
    entry is -1: the pool is full, or the table has no room).

    A sequence whose unfinished page could not be copied has lost that page's
    tokens. ``all_held=True`` says that no unfinished page was given back (no
    call here does that), so that one missing from a table is known to be lost:
    such a sequence comes back with the length of its full pages, without a
    page, counted as above, in this fork and in each that still finds it so.
    Without it lengths stay as they are, and a missing unfinished page counts
    as given back: the sequence goes on in a free page whose first tokens are
    another sequence's, for callers whose window hides them.

    A sequence's token is appended (at position seq_lens[r], which then grows
    by one) before it is forked again: a page taken for a token that never came
    is not found again by the next fork. A sequence that stays in the batch
    without going on, of length 0 too, has parent -1 for that reason. ``out``
    receives the new tables, for example the other half of a double buffer."""
    device = _state(block_tables, seq_lens, ref_counts)
    _on_gpu_i32(parents, "parents", 1)
    if parents.numel() != seq_lens.numel() or parents.device != device:
        raise ValueError("parents must hold one row number per sequence, on the same GPU")
    ptr, layer_stride, layers, page_stride, page_bytes, pages = _pool(kv_pool, ref_counts)
    rows, width = block_tables.shape
    if out is None:
        out = block_tables.new_empty((rows, width))
    elif out.shape != block_tables.shape or out.device != device:
        raise ValueError("out must have block_tables' shape and device")
    else:
        _on_gpu_i32(out, "out", 2)
        span = 4 * ((rows - 1) * _row_stride(block_tables) + width)
        out_span = 4 * ((rows - 1) * _row_stride(out) + width)
        if rows and width and (out.data_ptr() < block_tables.data_ptr() + span
                               and block_tables.data_ptr() < out.data_ptr() + out_span):
            raise ValueError("out must not share memory with block_tables")
    # lengths and counts that go back, then the kernels' scratch
    lens, counts, scratch = ref_counts.new_empty(4 * rows + 3).split_with_sizes((rows, 3, 3 * rows))
    with _device_guard(device):
        lib = _lib.load()
        _lib.check((lib.pa_fork_held_sequences if all_held else lib.pa_fork_sequences)(
            ptr, layer_stride, layers, page_stride, page_bytes, pages, block_tables.data_ptr(),
            _row_stride(block_tables), width, seq_lens.data_ptr(), parents.data_ptr(), rows,
            _page_size(kv_pool, kv_layout), ref_counts.data_ptr(), out.data_ptr(), _row_stride(out),
            lens.data_ptr(), counts.data_ptr(), scratch.data_ptr(), _stream()), "fork_sequences")
        _after("fork_sequences")
    return out, lens, counts


def compact_pages(kv_pool: torch.Tensor, block_tables: torch.Tensor, seq_lens: torch.Tensor,
                  ref_counts: torch.Tensor, kv_layout: str = "HND"
                  ) -> Tuple[torch.Tensor, torch.Tensor]:
    """Moves the live pages (count > 0) to the front of the pool, in place:
    with n of them, the k-th live page at or past n goes to the k-th free page
    before n (all layers); ``ref_counts`` and the entries of ``block_tables``
    follow. Returns (remap, counts): remap [pages] is each live page's new
    number, -1 for free ones, for holders outside the tables (a prefix
    cache); counts: live pages, pages moved, errors (entries whose page
    nobody holds, which stay, and rows whose length is past the table)."""
    device = _state(block_tables, seq_lens, ref_counts)
    ptr, layer_stride, layers, page_stride, page_bytes, pages = _pool(kv_pool, ref_counts)
    remap, counts = ref_counts.new_empty(pages), ref_counts.new_empty(3)
    scratch = ref_counts.new_empty(pages + 2)
    with _device_guard(device):
        _lib.check(_lib.load().pa_compact_pages(
            ptr, layer_stride, layers, page_stride, page_bytes, pages, block_tables.data_ptr(),
            _row_stride(block_tables), block_tables.size(1), seq_lens.data_ptr(),
            seq_lens.numel(), _page_size(kv_pool, kv_layout), ref_counts.data_ptr(),
            remap.data_ptr(), counts.data_ptr(), scratch.data_ptr(), _stream()), "compact_pages")
        _after("compact_pages")
    return remap, counts
