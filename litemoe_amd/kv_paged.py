"""The paged cache's store, read-back and eviction (``lm_paged_rotate_write``,
``lm_paged_read``, ``lm_kv_evict``) for :class:`~litemoe_amd.cache.PagedKVCache`.

Keys and values lie in pages of a pool, and a table names each row's pages, so
that a row takes memory by its own length, rows may share the pages of a common
beginning, and an eviction gives pages back. The reference's cache is one page of
the whole capacity per row (litemoe/cache.py:7-20, flash_decode.py:10-12).
"""
import torch

from . import _lib
from .kv_quant import per_row

PAGES = frozenset(1 << s for s in range(4, 17))  # positions of a page
HEAD_DIMS = (64, 128)
IN_PLACE = 12288  # positions of a row whose weights an eviction may write where it reads them


def check_layer(k, v, table):
    """The device index of one layer's buffers ``k, v [P, H, page, D]``, ``table [B, W]``."""
    index, shape = k.get_device(), k.shape
    if index < 0 or v.get_device() != index or table.get_device() != index:
        _lib.require_cuda(k, v, table, what="paged KV cache")
        raise ValueError("Paged KV cache layers must share one device")
    if len(shape) != 4 or v.shape != shape or shape[2] not in PAGES or shape[3] not in HEAD_DIMS:
        raise ValueError("Paged KV cache layers are k, v [P, H, page, D], page a power of two from 16 to 65536, "
                         "D 64 or 128")
    if k.dtype != torch.bfloat16 or v.dtype != torch.bfloat16 or not k.is_contiguous() or not v.is_contiguous():
        raise ValueError("Paged KV cache layers must be contiguous BF16")
    if table.dtype != torch.int32 or table.dim() != 2 or not table.is_contiguous():
        check_table(table)
    return index


def check_table(table, rows=None):
    if table.dtype != torch.int32 or table.dim() != 2 or not table.is_contiguous() or not table.shape[1]:
        raise ValueError("A page table is contiguous int32 [rows, pages of a row]")
    if rows is not None and table.shape[0] != rows:
        raise ValueError("The page table needs one line per row")


def places(t, rows, index, what):
    """``t``, a place in the cache per row, as the kernels take it: int64 or int32."""
    return per_row(t, rows, torch.int32 if t.dtype == torch.int32 else torch.int64, index, what)


def view(x, rows, heads):
    """``x [rows, heads, D]`` as the kernels take it, contiguous channels, rows and heads
    that start at 16 bytes (a copy where it is not so), and its pointer and strides."""
    at, (s0, s1, s2) = x.data_ptr(), x.stride()
    # of a single row or head the stride says nothing
    s0, s1 = s0 if rows > 1 else 0, s1 if heads > 1 else 0
    if s2 != 1 or s0 % 8 or s1 % 8 or at % 16:
        x = x.clone(memory_format=torch.contiguous_format)
        return x, (x.data_ptr(), heads * x.shape[2], x.shape[2])
    return x, (at, s0, s1)


def write(cache, layer, k, v, positions, active, slots):
    """Store ``k[row, h, 0, :]`` at position ``positions[row]`` of ``slots[row]`` for
    active rows (same for v), as :func:`kv_write.write`. ``k, v [rows, H, 1, D]``
    bf16 with any strides; ``active`` may be None (every row). Rows out of range or
    without a page there are skipped. One row per target."""
    kc, vc, table = cache.layer(layer)
    index = check_layer(kc, vc, table)
    pages, heads, page, dim = kc.shape
    if k.dim() != 4 or k.shape[1:] != (heads, 1, dim) or v.shape != k.shape:
        raise ValueError("KV write takes k, v [rows, H, 1, D] of the cache's heads")
    if k.dtype != torch.bfloat16 or v.dtype != torch.bfloat16:
        raise ValueError("The paged KV write supports BF16")
    if k.get_device() != index or v.get_device() != index:
        raise ValueError("KV write tensors must be on the cache's device")
    rows = k.shape[0]
    at = places(positions, rows, index, "positions")
    slots = per_row(slots, rows, torch.int64, index, "slots")
    # held here until the launch: memory given back before it is the next copy's
    active = None if active is None else per_row(active, rows, torch.bool, index, "active")
    (k, k_view), (v, v_view) = view(k[:, :, 0], rows, heads), view(v[:, :, 0], rows, heads)
    _lib.call_struct(index, "lm_paged_rotate_write", 0, 0, 0, *k_view, *v_view, 0, 0, 0, 0, 0, 0, at.data_ptr(),
                     at.dtype == torch.int32, 0 if active is None else active.data_ptr(), slots.data_ptr(),
                     0, 0, 0, 0, 0, 0, kc.data_ptr(), vc.data_ptr(), table.data_ptr(), table.shape[0], table.shape[1],
                     pages, page, rows, 0, heads, dim)


def read(cache, layer, positions, slots):
    """What the cache holds at ``(slots[row], h, positions[row])``: ``k, v [rows, H,
    1, D]``, the layout :func:`write` takes. Rows out of range or without a page
    there give zeros."""
    kc, vc, table = cache.layer(layer)
    index = check_layer(kc, vc, table)
    pages, heads, page, dim = kc.shape
    rows = positions.numel()
    positions = places(positions, rows, index, "positions")
    slots = per_row(slots, rows, torch.int64, index, "slots")
    k = kc.new_empty((rows, heads, 1, dim))
    v = torch.empty_like(k)
    _lib.call_struct(index, "lm_paged_read", kc.data_ptr(), vc.data_ptr(), table.data_ptr(), table.shape[0],
                     table.shape[1], pages, page, positions.data_ptr(), positions.dtype == torch.int32, slots.data_ptr(),
                     rows, heads, dim, k.data_ptr(), v.data_ptr())
    return k, v


def evict(cache, weights, used, keep, recent, target, table=None, weights_out=None):
    """Of each row's ``used[b]`` positions, per layer and KV head, the ``recent`` last
    and the heaviest of the others by ``weights [L, B, H, W * page]`` (fp32; see
    :meth:`flash_decode.PagedFlashDecode.__call__`) are copied, ``keep`` in all and in
    their order, to the pages that ``target [B, W']`` names. Returns the weights of
    what stays (then zeros; in ``weights_out``, which may be ``weights``, if given), the
    positions kept ``[L, B, H, keep]`` (int32, then -1) and the rows' new ``used``.

    Of equal weights the first stays; a NaN counts as the heaviest. A position that has
    no page stays as zeros, as it is read. ``table`` is the rows' present table (the
    cache's own unless given). Pages of ``target`` must not be in it: the rows' present
    pages are read and not written, so another row may share them.
    :meth:`PagedKVCache.evict` takes care of both and moves the cache's table."""
    k, v = cache.k, cache.v
    table = cache.table if table is None else table
    layers, pages, heads, page, dim = k.shape
    index = k.get_device()
    if index < 0 or table.get_device() != index:
        _lib.require_cuda(k, table, what="paged KV cache")
        raise ValueError("Eviction's tables and weights must be on the cache's device")
    check_table(table)
    rows, width = table.shape
    check_table(target, rows)
    if target.get_device() != index or weights.get_device() != index:
        raise ValueError("Eviction's tables and weights must be on the cache's device")
    shape = (layers, rows, heads, width * page)
    for w in (weights,) if weights_out is None or weights_out is weights else (weights, weights_out):
        if w.dtype is not torch.float32 or w.shape != shape or not w.is_contiguous() or w.get_device() != index:
            raise ValueError("Weights must be contiguous fp32 [L, B, H, positions of a row] on the cache's device")
    keep, recent = int(keep), int(recent)
    if not 1 <= keep <= width * page or not 0 <= recent <= keep:
        raise ValueError("Eviction keeps 1 to all positions of a row, and at most that many recent ones")
    used = per_row(used, rows, torch.int32, index, "used")
    out = torch.empty_like(weights) if weights_out is None else weights_out
    if out.data_ptr() == weights.data_ptr() and width * page > IN_PLACE:
        weights = weights.clone()
    kept, left = table.new_empty((layers, rows, heads, keep)), table.new_empty(rows)
    _lib.call_struct(index, "lm_kv_evict", k.data_ptr(), v.data_ptr(), table.data_ptr(), target.data_ptr(), width,
                     target.shape[1], pages, page, used.data_ptr(), weights.data_ptr(), layers, rows, heads, dim, keep,
                     recent, out.data_ptr(), kept.data_ptr(), left.data_ptr())
    return out, kept, left
