"""fxlm.paged: a KV cache in pages, besides its attention (fxlm.attention.paged_attention).

The cache is a pool of pages of P rows in every layer, (N, P, Hkv, Dh); a row of a batch (a request, a
beam) has the pages that its line of a table names, one after the other, and takes more as it grows.
Rows may hold a page together: ``uses`` counts the rows that hold each, and a page without uses is
free.  The reference has no cache (its ml/fxlm/sample.py:62-73 re-runs the context for every token).
All of it is inference, runs on torch's current stream, reads no device value on the host and can be
captured in a graph.
"""
import torch

from fxgpu.abi import host

from .attention import check_page
from .speculative import _taken

MOST_ROWS = 8192   # of a table


def extend_pages(table, lens, add, uses, page, most=1, cache=None):
    """Give each row pages for the tokens that it is about to add.

    table (R, M) int32 cuda, R <= 8192: row r's pages, of which ceil(lens[r] / page) are in use; lens, add (R,)
    int32 cuda: its tokens and the new ones, at most `most` of them (more count as `most`); uses (N,)
    int32 cuda: the rows that hold each page.  page: rows of a page, a power of two from 16 to 1024.
    Free pages are taken from the lowest on, in the order of the rows; table and uses are changed in place.
    cache, a list of (k, v) pools (N, page, Hkv, Dh) bf16: where a row's last page is not full and other
    rows hold it too, the row gets one of its own with the same rows in it, in every pool; if all of the
    holders are about to write there, the one with the most tokens keeps it, the lowest of equals (so that
    nothing of a holder that is refused a page is written over).  Without cache such a row gets nothing.

    Returns slots (R, most) int64, the place page * P + row of each new token in the pools' rows, -1
    behind a row's own, and the new lengths (R,) int32.  A row that cannot have all of its pages (the
    pool's are used up by it and the rows before it that want some, or they exceed M, or its last page is
    no page of the pool) gets nothing: its slots are -1, its length stays.
    """
    r = host.extend_pages(table, lens, add, uses, int(page), int(most), cache)
    if r is None:
        _check_tables(table, page, uses, lens=lens, add=add)
        if not 1 <= int(most) < 2 ** 31:
            raise ValueError(f"most={most} must be positive")
        if cache is not None:
            pools = [t for kv in cache for t in kv]
            if not pools:
                raise ValueError("cache holds no tensors")
            for t in pools:
                _check_pool(t, pools[0].shape)
            if pools[0].shape[0] != uses.numel() or pools[0].shape[1] != page:
                raise ValueError(f"pools {tuple(pools[0].shape)} of {uses.numel()} pages of {page} rows")
        r = host.extend_pages(table, lens.contiguous(), add.contiguous(), uses, int(page), int(most), cache)
    return _taken(r, "extend_pages")


def store_pages(k, v, slots, k_pages, v_pages):
    """Write rows into pools: k, v (R, T, Hkv, Dh) bf16 to rows slots (R, T) int64 cuda (extend_pages') of
    k_pages, v_pages (N, P, Hkv, Dh) bf16, in place.  A slot that is none of the N * P is passed over; no
    slot may be there twice."""
    if not host.store_pages(k, v, slots, k_pages, v_pages):
        if k.dim() != 4 or v.shape != k.shape or min(k.shape) < 1:
            raise ValueError(f"k and v must share one shape (R, T, Hkv, Dh): {tuple(k.shape)} {tuple(v.shape)}")
        for nm, t in (("k", k), ("v", v)):
            if t.dtype != torch.bfloat16 or not t.is_cuda:
                raise TypeError(f"{nm} must be a bfloat16 cuda tensor")
            if t.stride(-1) != 1 or any(x % 8 for x in t.stride()[:-1]) or t.data_ptr() % 16:
                raise ValueError(f"{nm}: last dim must be contiguous, other strides multiples of 8 elements and the base 16-byte aligned")
        for t in (k_pages, v_pages):
            _check_pool(t, k_pages.shape)
        if k_pages.shape[2:] != k.shape[2:]:
            raise ValueError(f"rows {tuple(k.shape)} do not match the pools {tuple(k_pages.shape)}")
        if slots.dtype != torch.int64 or not slots.is_cuda or slots.shape != k.shape[:2]:
            raise TypeError(f"slots must be an int64 cuda tensor of shape {tuple(k.shape[:2])}")
        raise ValueError("store_pages: tensors of a layout or size that it does not take")


def reorder_pages(table, lens, parents, uses, page):
    """Let each row go on from another: row r of table (R, M) int32 cuda, R <= 8192, takes the pages of row
    parents[r] (R,) int32 cuda, beside whoever else does, or ends where that is no row (-1).  lens (R,)
    int32 cuda: the rows' tokens; uses (N,) int32 cuda is brought up to date.  In place; entries behind a
    row's new pages keep what they held.  Returns the rows' new lengths (R,) int32."""
    r = host.reorder_pages(table, lens, parents, uses, int(page))
    if r is None:
        _check_tables(table, page, uses, lens=lens, parents=parents)
        r = host.reorder_pages(table, lens.contiguous(), parents.contiguous(), uses, int(page))
    return _taken(r, "reorder_pages")


def _check_tables(table, page, uses, **rows):
    """Raise for a table and its companions that the functions here do not take."""
    check_page(page)
    if table.dtype != torch.int32 or not table.is_cuda or table.dim() != 2:
        raise TypeError("table must be an int32 cuda tensor (R, M)")
    R, M = table.shape
    if not 1 <= R <= MOST_ROWS or M < 1:
        raise ValueError(f"table {tuple(table.shape)}: 1 to {MOST_ROWS} rows of a page at least")
    if table.stride(1) != 1 and M > 1 or R > 1 and table.stride(0) < M:
        raise ValueError("table: last dim must be contiguous, and no two rows may overlap")
    for nm, t in rows.items():
        if t.dtype != torch.int32 or not t.is_cuda or tuple(t.shape) != (R,):
            raise TypeError(f"{nm} must be an int32 cuda tensor of shape ({R},)")
    if uses.dtype != torch.int32 or not uses.is_cuda or uses.dim() != 1 or not uses.is_contiguous():
        raise TypeError("uses must be a contiguous int32 cuda tensor (N,)")
    if uses.numel() < 1:
        raise ValueError("uses: a page at least")


def _check_pool(t, shape):
    """Raise for what is no pool of pages of this shape."""
    if t.dtype != torch.bfloat16 or not t.is_cuda:
        raise TypeError("pools must be bfloat16 cuda tensors")
    if t.dim() != 4 or t.shape != shape or min(t.shape) < 1 or t.shape[3] % 8:
        raise ValueError(f"pools must share one shape (N, P, Hkv, Dh), Dh a multiple of 8: {tuple(t.shape)}")
    check_page(t.shape[1])
    if any(st == 0 and n > 1 for st, n in zip(t.stride(), t.shape)):
        raise ValueError("an expanded pool cannot be written to")
    if t.stride(-1) != 1 or any(x % 8 for x in t.stride()[:-1]) or t.data_ptr() % 16:
        raise ValueError("pools: last dim must be contiguous, other strides multiples of 8 elements and the base 16-byte aligned")


class PagedCache:
    """A paged cache for `rows` rows of a batch: pools of `pages` pages of `page` rows for each of `layers`
    layers, the table, the rows' lengths and the pages' uses.  All rows begin without tokens.

    ``extend(add, most)`` gives rows pages for their next tokens and returns the slots; ``reorder(parents)``
    lets rows go on from others or end.  Both change ``table``, ``lens`` and ``uses`` in place, so that a
    graph can hold them (one captured before the first ``reorder`` copies no pages: rows that would need
    a copy get nothing there).  ``table`` has room for `width` pages a row."""

    def __init__(self, rows, pages, page, width, layers, heads, head_dim, device):
        check_page(page)
        if min(rows, pages, width, layers) < 1 or rows > MOST_ROWS:
            raise ValueError(f"a paged cache of {rows} rows (1 to {MOST_ROWS}), {pages} pages, {width} a row, {layers} layers")
        self.page = page
        # a page's rows of one head lie together
        self.pools = torch.zeros(layers, 2, pages, heads, page, head_dim, device=device, dtype=torch.bfloat16).transpose(3, 4)
        self.kv = [(p[0], p[1]) for p in self.pools]
        self.table = torch.full((rows, width), -1, device=device, dtype=torch.int32)
        self.lens = torch.zeros(rows, device=device, dtype=torch.int32)
        self.uses = torch.zeros(pages, device=device, dtype=torch.int32)
        self.shared = False   # whether rows may hold pages together: a row went on from another

    def extend(self, add, most=1):
        """extend_pages for add (R,) int32 new tokens a row; returns the slots (R, most) int64."""
        slots, lens = extend_pages(self.table, self.lens, add, self.uses, self.page, most, self.kv if self.shared else None)
        self.lens.copy_(lens)
        return slots

    def reorder(self, parents):
        """reorder_pages for parents (R,) int32."""
        self.lens.copy_(reorder_pages(self.table, self.lens, parents, self.uses, self.page))
        self.shared = True

    def end(self, rows=None):
        """Rows (an index tensor, all by default) give their pages back."""
        parents = torch.arange(self.lens.numel(), device=self.lens.device, dtype=torch.int32)
        parents[slice(None) if rows is None else rows] = -1
        self.lens.copy_(reorder_pages(self.table, self.lens, parents, self.uses, self.page))
