"""Pages of a cache: who holds them, on the device.

``block_table [rows, max_pages] int32`` (-1: no page), ``seq_lens [rows] int32`` and
``refs [n_pages] int32``, the number of table entries that hold each page.  A page is free
where its count is 0, and allocation takes the lowest free pages, so the state after a call
is a function of the state before it.  ``tensors`` is every tensor whose pages the table
names, as any iterable of ``[n_pages, ...]``: the K and V pools of all layers and, for fp8, their
scales; they need not be contiguous.

Calls launch on the current stream of the tensors' device, never synchronise and can be
captured.  One state's calls must be ordered (one stream).
"""

import ctypes
import functools
import operator
import struct

import torch

from . import _native as N
from .ops import workspace_tensor
from .prompt import check_ints, device_of, launch


_TAIL_BYTES = ctypes.sizeof(N.PageTensor) - 8


@functools.lru_cache(maxsize=512)
def _page_layout(shape, stride, itemsize):
    """``(page_stride, outer_stride, inner_stride, n_outer, n_inner, run_bytes, word)`` of a
    tensor's pages, in bytes: its dimensions behind the first, neighbours in memory joined."""
    runs = sorted((s, n) for n, s in zip(shape[1:], stride[1:]) if n != 1)
    if any(s == 0 for s, _ in runs) or 0 in shape[1:]:
        raise ValueError("page tensors must not be empty or expanded")
    joined = [(1, 1)]
    for s, n in runs:
        if s == joined[-1][0] * joined[-1][1]:
            joined[-1] = (joined[-1][0], joined[-1][1] * n)
        elif s < joined[-1][0] * joined[-1][1]:
            raise ValueError("page tensors must not overlap themselves")
        else:
            joined.append((s, n))
    if len(joined) > 3:
        raise ValueError("a page's elements must lie in at most two levels of contiguous runs")
    joined += [(0, 1)] * (3 - len(joined))
    (_, run), (inner, n_inner), (outer, n_outer) = joined
    if shape[0] > 1 and stride[0] < 1:
        raise ValueError("page tensors must not be empty or expanded")
    size = (stride[0] * itemsize, outer * itemsize, inner * itemsize, run * itemsize)
    word = 16 if all(x % 16 == 0 for x in size) else 4
    if any(x % word for x in size):
        raise ValueError("pages must be made of multiples of 4 bytes")
    return size[0], size[1], size[2], n_outer, n_inner, size[3], word


@functools.lru_cache(maxsize=512)
def _struct_tail(shape, stride, dtype, word):
    """A ``PageTensor``'s bytes behind its pointer, with words of ``word`` bytes if they fit."""
    lay = _page_layout(shape, stride, torch.empty((), dtype=dtype).element_size())
    return bytes(N.PageTensor(None, *lay[:6], min(lay[6], word)))[8:]


def _page_tensors(tensors, n_pages, ref):
    """C array of page tensors; ``n_pages`` None takes the first tensor's."""
    tensors = tuple(tensors)  # (walked twice: an iterator would be at its end)
    dev, at = ref.get_device(), [t.data_ptr() for t in tensors]
    if not at:
        return None, 0, 0
    low = functools.reduce(operator.or_, at) & 15
    if low & 3:
        raise ValueError("pages must be 4-byte aligned")
    parts, known, last, tail = [], [], None, None
    for t, p in zip(tensors, at):
        layout = (t.shape, t.stride(), t.dtype)
        if layout != last or low:  # (a model's pools are alike)
            for last, tail in known if not low else ():
                if layout == last:
                    break
            else:
                shape = layout[0]
                if n_pages is None:
                    n_pages = shape[0] if len(shape) else 0
                if len(shape) < 2 or shape[0] != n_pages:
                    raise ValueError(f"page tensors must be [n_pages, ...] with {n_pages} pages")
                last, tail = layout, _struct_tail(*layout, 4 if p & 15 else 16)
                known.append((last, tail))
        if t.get_device() != dev:
            raise ValueError(f"page tensors must be on {ref.device}, got {t.device}")
        parts += p, tail
    n = len(at)
    return (N.PageTensor * n).from_buffer_copy(struct.pack(f"Q{_TAIL_BYTES}s" * n, *parts)), n, n_pages


def _state(block_table, seq_lens, refs, page_size, *others):
    device_of(refs, block_table, seq_lens, *others)
    if block_table.dtype != torch.int32 or block_table.dim() != 2:
        raise ValueError("block_table must be int32 [rows, max_pages] with contiguous rows")
    (rows, cols), (stride, inner) = block_table.shape, block_table.stride()
    if cols > 1 and inner != 1:
        raise ValueError("block_table must be int32 [rows, max_pages] with contiguous rows")
    if rows <= 1:
        stride = cols
    elif stride < cols:
        raise ValueError("block_table rows must not overlap")
    n_pages = check_ints(refs, "refs")
    if seq_lens is not None:
        check_ints(seq_lens, "seq_lens", rows)
    if page_size <= 0:
        raise ValueError("page_size must be positive")
    return N.PageState(block_table.data_ptr(), stride, rows, cols, None if seq_lens is None else seq_lens.data_ptr(),
                       refs.data_ptr(), n_pages, page_size)


def copy_pages(tensors, src, dst):
    """Copy page ``src[i]`` of every tensor to page ``dst[i]`` (``[n] int32`` on the device),
    all tensors in one launch.  Pages that do not exist are skipped; no page may be twice in
    ``dst``, or in ``src`` and in ``dst``."""
    device_of(src, dst)
    count = check_ints(src, "src")
    check_ints(dst, "dst", count)
    desc, n, n_pages = _page_tensors(tensors, None, src)
    launch(N.lib().ia_copy_pages, src, desc, n, src.data_ptr(), dst.data_ptr(), count, n_pages)


def fork_sequences(tensors, block_table, seq_lens, refs, src_rows, dst_rows, *, page_size, workspace=None):
    """Make row ``dst_rows[i]`` a continuation of row ``src_rows[i]`` (``[n] int32`` on the
    device): whole pages are shared (``refs`` rise), the page the source's last tokens partly
    fill is copied in every tensor to the lowest free page, and the length is taken over.
    Both rows can then be appended to.  Returns ``ok [n] int32``: 1, or 0 and the row as it
    was where a row does not exist, ``dst_rows[i]`` is not empty (``free_sequences``) or
    listed before, ``src_rows[i]`` is in ``dst_rows`` or its last page is not mapped, or no
    page is free.  At most 8192 forks a call."""
    state = _state(block_table, seq_lens, refs, page_size, src_rows, dst_rows)
    desc, n_t, _ = _page_tensors(tensors, state.n_pages, refs)
    n = check_ints(src_rows, "src_rows")
    check_ints(dst_rows, "dst_rows", n)
    ok = torch.empty_like(src_rows)
    lib = N.lib()
    ws = workspace_tensor(workspace, ("fork_scratch", n), (max(lib.ia_fork_workspace_size(n), 4),), device=refs.device,
                          dtype=torch.uint8)
    launch(lib.ia_fork_sequences, refs, state, desc, n_t, src_rows.data_ptr(), dst_rows.data_ptr(), n, ok.data_ptr(),
           ws.data_ptr(), ws.numel())
    return ok


def free_sequences(block_table, seq_lens, refs, rows):
    """Rows ``rows`` (``[n] int32`` on the device) give up their pages: ``refs`` fall, table
    entries become -1, lengths 0.  A row listed twice is freed once; rows that do not exist
    are skipped."""
    state = _state(block_table, seq_lens, refs, 1, rows)
    launch(N.lib().ia_free_sequences, refs, state, rows.data_ptr(), check_ints(rows, "rows"))


def reserve_pages(block_table, seq_lens, refs, new_tokens, *, page_size, workspace=None):
    """Give every row the pages its next ``new_tokens[row]`` tokens reach (``[rows] int32`` on
    the device; 0: none), the lowest free ones, rows in order.  Returns ``ok [rows] int32``:
    1, or 0 and the row as it was where its table row is too short or the pages left do not
    cover it."""
    state = _state(block_table, seq_lens, refs, page_size, new_tokens)
    rows = check_ints(new_tokens, "new_tokens", state.rows)
    lib = N.lib()
    ok = torch.empty_like(new_tokens)
    need = max(lib.ia_reserve_workspace_size(rows, state.n_pages), 4)
    ws = workspace_tensor(workspace, ("reserve_scratch", need), (need,), device=refs.device, dtype=torch.uint8)
    launch(lib.ia_reserve_pages, refs, state, new_tokens.data_ptr(), ok.data_ptr(), ws.data_ptr(), ws.numel())
    return ok


def reorder_sequences(tensors, block_table, seq_lens, refs, parents, *, page_size, workspace=None):
    """Every row becomes what row ``parents[row]`` (``[rows] int32`` on the device) was, all at
    once: beams that follow their parents.  Of the rows with one parent, the parent itself,
    else the lowest, takes its pages over as they are; the others share its whole pages
    (``refs`` rise) and get a copy, in every tensor, of the page its last tokens partly fill, in
    the lowest free page, rows in order.  Pages that no row holds any more are free, for the
    copies too.  A parent outside the rows (-1) leaves the row empty.  Rows that are no beams
    are their own parents: nothing of them is touched.  Returns ``ok [rows] int32``: 1, or 0 and
    the row empty where the partly filled page is not mapped, the length does not fit the
    table or no page is free.  At most 8192 rows.  What else follows rows (block summaries,
    sequence scales) is indexed with ``parents`` by the caller."""
    state = _state(block_table, seq_lens, refs, page_size, parents)
    desc, n_t, _ = _page_tensors(tensors, state.n_pages, refs)
    check_ints(parents, "parents", state.rows)
    ok = torch.empty_like(parents)
    lib = N.lib()
    need = max(lib.ia_reorder_workspace_size(state.rows, state.cols), 4)
    ws = workspace_tensor(workspace, ("reorder_scratch", state.rows, state.cols), (need,), device=refs.device, dtype=torch.uint8, zero=True)
    launch(lib.ia_reorder_sequences, refs, state, desc, n_t, parents.data_ptr(), ok.data_ptr(), ws.data_ptr(),
           ws.numel())
    return ok


def compact_pages(tensors, block_table, refs, *, workspace=None):
    """Move the live pages to the front of the pools: of ``n_live`` held pages, those at or
    past ``n_live`` move, in ascending order, to the free pages before it; ``block_table`` and
    ``refs`` follow.  Returns ``n_live`` (``[1] int32`` on the device): every page from there
    on is free, so the pools can be cut or lent out.  Whatever else names pages (fp8
    ``sequence_scales``, copies of the table) has to be rebuilt."""
    state = _state(block_table, None, refs, 1)
    desc, n_t, _ = _page_tensors(tensors, state.n_pages, refs)
    lib = N.lib()
    n_live = torch.empty(1, device=refs.device, dtype=torch.int32)
    need = lib.ia_compact_workspace_size(state.n_pages)
    ws = workspace_tensor(workspace, ("compact_scratch", need), (need,), device=refs.device, dtype=torch.uint8)
    launch(lib.ia_compact_pages, refs, state, desc, n_t, n_live.data_ptr(), ws.data_ptr(), ws.numel())
    return n_live
