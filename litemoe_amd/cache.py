"""Contiguous rank-local KV cache ``[L, B, Hkv, C, D]`` (litemoe/cache.py:7-55).

The layout is the reference's: row b of the batch owns cache page b, a whole
``capacity``-long sequence per KV head. Writes go through the masked gfx950
store (one writer per row, head and channel).

:class:`QuantKVCache` has the same interface over a cache of 4 or 8 bits per
element (:mod:`litemoe_amd.kv_quant`); :class:`PagedKVCache` over pages of a
pool (:mod:`litemoe_amd.kv_paged`)."""
from typing import NamedTuple

import torch

from . import kv_paged, kv_quant, kv_write


class KVCache:
    def __init__(self, cfg, batch, capacity, device, dtype):
        self.capacity = capacity
        h, d = cfg.num_key_value_heads, cfg.hidden_size // cfg.num_attention_heads
        shape = (cfg.num_hidden_layers, batch, h, capacity, d)
        self.k = torch.zeros(shape, dtype=dtype, device=device)
        self.v = torch.zeros_like(self.k)
        self.keys = torch.arange(capacity, device=device)
        self.slots = torch.arange(batch, device=device)

    def reset(self):
        self.k.zero_()
        self.v.zero_()

    def prefill(self, layer, slot, k, v, valid):
        """Store a prefill's ``k, v`` and return ``(k, v, mask)``
        (litemoe/cache.py:21-33). ``slot`` a :class:`PackedPrefill`: ``k, v
        [1, H, T, D]`` go to ``(slot.slots[t], h, slot.positions[t])`` and the
        mask is None. ``slot`` an int or a slice: ``k, v [b, H, s, D]`` times
        ``valid [b, s]`` go to positions ``0 .. s-1`` of rows ``slot``; the
        mask ``[b, 1, s, s]`` is causal over valid keys, and a padding query
        sees key 0 only."""
        from .packed import PackedPrefill
        if isinstance(slot, PackedPrefill):
            tokens = k.shape[2]
            kv_write.write(self, layer, k[0].transpose(0, 1).unsqueeze(2), v[0].transpose(0, 1).unsqueeze(2),
                           slot.positions,
                           torch.ones(tokens, dtype=torch.bool, device=k.device), slot.slots)
            return k, v, None
        s = k.shape[2]
        rows = slot if isinstance(slot, slice) else slice(slot, slot + 1)
        keep = valid[:, None, :, None]
        self.k[layer, rows, :, :s].copy_(torch.where(keep, k, torch.zeros((), dtype=k.dtype, device=k.device)))
        self.v[layer, rows, :, :s].copy_(torch.where(keep, v, torch.zeros((), dtype=v.dtype, device=v.device)))
        pos = torch.arange(s, device=k.device)
        mask = (pos[:, None] >= pos[None, :])[None, None] & valid[:, None, None, :]
        mask = torch.where(valid[:, None, :, None], mask, (pos == 0)[None, None, None, :])
        return k, v, mask

    def decode(self, layer, k, v, lengths, active):
        """Masked store of one decode step's ``k, v [B, H, 1, D]`` at
        ``where(active, lengths, 0)``; returns the layer's cache and the key
        mask ``[B, 1, 1, C]`` (keys below ``lengths + 1``, key 0 for inactive
        rows), litemoe/cache.py:42-47."""
        pos = torch.where(active, lengths, 0)
        self.write(layer, k, v, pos, active)
        mask = self.keys[None, :] < (lengths + 1)[:, None]
        mask = torch.where(active[:, None], mask, self.keys[None, :] == 0)
        return self.k[layer], self.v[layer], mask[:, None, None, :]

    def write(self, layer, k, v, pos, active, slots=None):
        """Masked store of ``k, v [rows, H, 1, D]`` at ``(slots, h, pos)``
        (cache.py:50-55 -> kv_write.py:23-29)."""
        return kv_write.write(self, layer, k, v, pos, active, self.slots if slots is None else slots)


FusedKVCache = KVCache


class QuantLayer(NamedTuple):
    """One layer of a :class:`QuantKVCache`, in the order the attention takes it."""
    k: torch.Tensor
    v: torch.Tensor
    scales: torch.Tensor


def _buffer(name):
    """A buffer of a :class:`QuantKVCache`: another of the same kind may take its place, and
    the views of the layers are then made anew."""
    def get(self):
        return self.__dict__[name]

    def put(self, t):
        held = self.__dict__.get(name)
        if held is not None and (t.shape != held.shape or t.dtype != held.dtype or t.device != held.device
                                 or not t.is_contiguous()):
            raise ValueError("Quantised KV buffers are replaced by contiguous ones of the same shape, type and device")
        self.__dict__[name] = t
        self._make_layers()
    return property(get, put)


class QuantKVCache:
    """A :class:`KVCache` whose elements take 4 or 8 bits: codes ``k, v [L, B,
    Hkv, C, 8*bits]`` and ``scales [L, B, Hkv, C, 4]``, uint8. The store
    quantises; attention reads the codes (``flash_decode.QuantFlashDecode``);
    :meth:`decode` and :func:`kv_quant.read` give back what they stand for.
    Prefill attends over its own unquantised keys and values, as
    :meth:`KVCache.prefill` returns them."""
    k, v, scales = _buffer("k"), _buffer("v"), _buffer("scales")

    def __init__(self, cfg, batch, capacity, device, dtype, bits=4):
        if dtype != torch.bfloat16:
            raise ValueError("A quantised KV cache stands for BF16 keys and values")
        if cfg.hidden_size // cfg.num_attention_heads != 64:
            raise ValueError("A quantised KV cache takes head_dim 64")
        self._bind(*self._buffers(cfg.num_hidden_layers, batch, cfg.num_key_value_heads, capacity, device, bits))

    @staticmethod
    def _buffers(layers, batch, heads, capacity, device, bits):
        if bits not in kv_quant.BITS:
            raise ValueError("A quantised KV cache holds 4 or 8 bits per element")
        shape = (layers, batch, heads, capacity)
        return [torch.zeros(*shape, n, dtype=torch.uint8, device=device) for n in (8 * bits, 8 * bits, 4)]

    @classmethod
    def empty(cls, layers, batch, heads, capacity, device, bits=4):
        """A cleared cache by its sizes, without a model's configuration."""
        return cls.over(*cls._buffers(layers, batch, heads, capacity, device, bits))

    @classmethod
    def over(cls, k, v, scales):
        """A cache over buffers that exist (a saved cache, memory that another
        cache owns): used in place, not copied."""
        if k.dim() != 5 or v.shape != k.shape or scales.shape != (*k.shape[:4], 4) or k.shape[4] not in (32, 64):
            raise ValueError("Quantised KV buffers are k, v [L, B, H, C, 8*bits] and scales [L, B, H, C, 4]")
        if any(t.dtype != torch.uint8 or not t.is_contiguous() or t.device != k.device for t in (k, v, scales)):
            raise ValueError("Quantised KV buffers must be contiguous uint8 on one device")
        cache = cls.__new__(cls)
        cache._bind(k, v, scales)
        return cache

    def _bind(self, k, v, scales):
        self.k, self.v, self.scales = k, v, scales
        self.bits, self.capacity = k.shape[4] // 8, k.shape[3]
        self.keys = torch.arange(self.capacity, device=k.device)
        self.slots = torch.arange(k.shape[1], device=k.device)

    def _make_layers(self):
        held = [self.__dict__.get(name) for name in QuantLayer._fields]
        self._layers = [] if any(t is None for t in held) else [QuantLayer(*buffers) for buffers in zip(*held)]

    def __setstate__(self, state):
        self.__dict__.update(state)
        self._make_layers()  # a copy's views are of its own buffers

    def layer(self, layer):
        """Layer ``layer``'s buffers, views of ``k``, ``v`` and ``scales`` made once."""
        return self._layers[layer]

    def reset(self):
        for t in (self.k, self.v, self.scales):
            t.zero_()

    def clear(self, row, start, stop):
        """Positions ``start .. stop-1`` of cache row ``row`` of every layer: zeros."""
        for t in (self.k, self.v, self.scales):
            t[:, row, :, start:stop].zero_()

    def prefill(self, layer, slot, k, v, valid):
        """:meth:`KVCache.prefill`: the store quantises, and the same ``(k, v,
        mask)`` come back."""
        from .packed import PackedPrefill
        if isinstance(slot, PackedPrefill):
            self.write(layer, k[0].transpose(0, 1).unsqueeze(2), v[0].transpose(0, 1).unsqueeze(2), slot.positions,
                       None, slot.slots)
            return k, v, None
        b, h, s, d = k.shape
        rows = self.slots[slot if isinstance(slot, slice) else slice(slot, slot + 1)]
        if s > self.capacity:
            raise ValueError("Prompt width exceeds the KV capacity")
        if rows.numel() != b:
            raise ValueError("Prefill slots must name one cache row per batch row")
        zero, keep = torch.zeros((), dtype=k.dtype, device=k.device), valid[:, None, :, None]
        pos = self.keys[:s]
        flat = [torch.where(keep, x, zero).transpose(1, 2).reshape(b * s, h, 1, d) for x in (k, v)]
        self.write(layer, *flat, pos.repeat(b), None, rows.repeat_interleave(s))
        mask = (pos[:, None] >= pos[None, :])[None, None] & valid[:, None, None, :]
        return k, v, torch.where(valid[:, None, :, None], mask, (pos == 0)[None, None, None, :])

    def decode(self, layer, k, v, lengths, active):
        """:meth:`KVCache.decode`, the layer's cache as the bf16 that it stands for."""
        pos = torch.where(active, lengths, 0)
        self.write(layer, k, v, pos, active)
        mask = self.keys[None, :] < (lengths + 1)[:, None]
        mask = torch.where(active[:, None], mask, self.keys[None, :] == 0)
        return *self.read(layer), mask[:, None, None, :]

    def write(self, layer, k, v, pos, active, slots=None):
        """Masked quantising store of ``k, v [rows, H, 1, 64]`` at ``(slots, h, pos)``."""
        return kv_quant.write(self, layer, k, v, pos, active, self.slots if slots is None else slots)

    def read(self, layer):
        """The whole layer as bf16 ``k, v [B, H, C, 64]``."""
        batch, capacity = self.slots.numel(), self.capacity
        sides = kv_quant.read(self, layer, self.keys.repeat(batch), self.slots.repeat_interleave(capacity))
        return tuple(x.view(batch, capacity, -1, 64).transpose(1, 2) for x in sides)


class PagedLayer(NamedTuple):
    """One layer of a :class:`PagedKVCache`, in the order the attention takes it."""
    k: torch.Tensor
    v: torch.Tensor
    table: torch.Tensor


class PagedKVCache:
    """A :class:`KVCache` whose rows take pages of a pool: ``k, v [L, P, Hkv, page,
    D]`` bf16, and ``table [B, W]`` (int32) names the pages of each row, -1 for none;
    position j of row b is page ``table[b, j // page]`` at ``j % page``, for all layers
    and heads. ``capacity`` (``W * page``) bounds a row, the pool's ``pages`` all of them
    together.

    A row has no pages until :meth:`reserve` gives it some; positions without a page are
    neither stored nor attended. :meth:`share` lets a row begin with another's pages,
    :meth:`evict` holds rows to a number of positions, :meth:`release` gives a row's
    pages back. These work on the host and change ``table`` in place, on the current
    stream: what was launched before on another stream has to be waited for first. A
    captured graph reads the table as it is when it replays."""

    def __init__(self, cfg, batch, capacity, device, dtype, page=64, pages=None):
        if dtype != torch.bfloat16:
            raise ValueError("A paged KV cache holds BF16 keys and values")
        dim = cfg.hidden_size // cfg.num_attention_heads
        self._bind(*self._buffers(cfg.num_hidden_layers, batch, cfg.num_key_value_heads, dim, capacity, device, page,
                                  pages))

    @staticmethod
    def _buffers(layers, batch, heads, dim, capacity, device, page, pages):
        if page not in kv_paged.PAGES or dim not in kv_paged.HEAD_DIMS:
            raise ValueError("A paged KV cache takes head_dim 64 or 128 and pages of a power of two from 16 to 65536 "
                             "positions")
        if min(layers, batch, heads, capacity) < 1 or (pages is not None and pages < 1):
            raise ValueError("A paged KV cache needs layers, rows, heads, positions and pages")
        width = -(-capacity // page)
        shape = (layers, batch * width if pages is None else pages, heads, page, dim)
        k = torch.zeros(shape, dtype=torch.bfloat16, device=device)
        return k, torch.zeros_like(k), torch.full((batch, width), -1, dtype=torch.int32, device=device)

    @classmethod
    def empty(cls, layers, batch, heads, dim, capacity, device, page=64, pages=None):
        """A cleared cache by its sizes, without a model's configuration."""
        cache = cls.__new__(cls)
        cache._bind(*cls._buffers(layers, batch, heads, dim, capacity, device, page, pages))
        return cache

    @classmethod
    def over(cls, k, v, table):
        """A cache over buffers that exist, used in place, not copied. Its pages are the
        caller's to hand out, through ``table``: :meth:`reserve`, :meth:`share`,
        :meth:`release` and :meth:`evict` are for caches that own their pool."""
        if k.dim() != 5 or v.shape != k.shape or k.shape[3] not in kv_paged.PAGES \
                or k.shape[4] not in kv_paged.HEAD_DIMS:
            raise ValueError("Paged KV buffers are k, v [L, P, H, page, D], page a power of two from 16 to 65536, D 64 "
                             "or 128")
        if any(t.dtype != torch.bfloat16 or not t.is_contiguous() or t.device != k.device for t in (k, v)):
            raise ValueError("Paged KV buffers must be contiguous BF16 on one device")
        kv_paged.check_table(table)
        if table.device != k.device:
            raise ValueError("Paged KV buffers must be on one device")
        cache = cls.__new__(cls)
        cache._bind(k, v, table)
        cache._free = None
        return cache

    def _bind(self, k, v, table):
        self._k, self._v, self._table = k, v, table
        self.page, self.capacity = k.shape[3], table.shape[1] * k.shape[3]
        self.keys = torch.arange(self.capacity, device=k.device)
        self.slots = torch.arange(table.shape[0], device=k.device)
        self._free = list(range(k.shape[1] - 1, -1, -1))  # taken from the end
        self._held = [[] for _ in range(table.shape[0])]  # pages of each row, in order
        self._rows_of = [0] * k.shape[1]                  # rows that hold each page
        self._make_layers()

    # the buffers are fixed: views of the layers are made once
    k = property(lambda self: self._k)
    v = property(lambda self: self._v)
    table = property(lambda self: self._table)

    def _make_layers(self):
        self._layers = [PagedLayer(k, v, self._table) for k, v in zip(self._k, self._v)]

    def __setstate__(self, state):
        self.__dict__.update(state)
        self._make_layers()  # a copy's views are of its own buffers

    def layer(self, layer):
        """Layer ``layer``'s keys and values, and the table."""
        return self._layers[layer]

    # -- pages ---------------------------------------------------------------
    def _owned(self):
        if self._free is None:
            raise ValueError("The pages of this cache are its caller's to hand out")

    def check_own(self, row, start, stop):
        """Raise ValueError where positions ``start .. stop-1`` of row ``row`` lie in a
        page that another row has too."""
        if self._free is None:  # the caller's pages
            return
        pages = self._held[self._row(row)]
        if start < stop and any(self._rows_of[page] > 1 for page in pages[start // self.page:-(-stop // self.page)]):
            raise ValueError("Pages that another row shares are not stored to")

    def _publish(self, rows):
        """The table's lines of ``rows`` from the lists on the host."""
        width = self._table.shape[1]
        lines = [self._held[row] + [-1] * (width - len(self._held[row])) for row in rows]
        index = torch.tensor(rows, device=self._table.device)
        self._table[index] = torch.tensor(lines, dtype=torch.int32).to(self._table.device)

    def _row(self, row):
        row = int(row)
        if not 0 <= row < len(self._held):
            raise ValueError("No such cache row")
        return row

    def _take(self, count):
        pages = [self._free.pop() for _ in range(count)]
        for page in pages:
            self._rows_of[page] = 1
        return pages

    def _drop(self, pages):
        for page in pages:
            self._rows_of[page] -= 1
            if not self._rows_of[page]:
                self._free.append(page)

    @property
    def free_pages(self):
        self._owned()
        return len(self._free)

    def held(self, row):
        """Positions that row ``row`` has pages for."""
        self._owned()
        return len(self._held[self._row(row)]) * self.page

    def reserve(self, rows, positions):
        """Pages for the first ``positions`` positions of ``rows`` (one or a list;
        ``positions`` one number or one per row), besides those that a row has. All or
        nothing: without enough free pages nothing changes and ValueError is raised."""
        self._owned()
        rows = [self._row(r) for r in (rows if isinstance(rows, (list, tuple)) else [rows])]
        if len(set(rows)) != len(rows):
            raise ValueError("Each cache row once")
        positions = list(positions) if isinstance(positions, (list, tuple)) else [positions] * len(rows)
        if len(positions) != len(rows) or any(not 0 <= p <= self.capacity for p in positions):
            raise ValueError("Positions of a row exceed the KV capacity")
        more = {row: max(0, -(-p // self.page) - len(self._held[row])) for row, p in zip(rows, positions)}
        if sum(more.values()) > len(self._free):
            raise ValueError(f"The KV pool has {len(self._free)} free pages, {sum(more.values())} are wanted")
        grown = [row for row in rows if more[row]]
        for row in grown:
            self._held[row] += self._take(more[row])
        if grown:
            self._publish(grown)

    def share(self, row, other, positions):
        """Row ``row``, which has no pages, begins with those of the first ``positions``
        positions of row ``other`` (a multiple of the page), which ``other`` has stored
        already. Both read them; neither may store there again: :meth:`clear`,
        :meth:`prefill` by rows and the model's prefills refuse it (:meth:`check_own`),
        a store by tensors of places is the caller's to keep out of them."""
        self._owned()
        row, other = self._row(row), self._row(other)
        if self._held[row] or row == other:
            raise ValueError("Only a row without pages can begin with another's")
        if positions < 0 or positions % self.page or positions > self.held(other):
            raise ValueError("Rows share whole pages that the other row has")
        self._held[row] = self._held[other][:positions // self.page]
        for page in self._held[row]:
            self._rows_of[page] += 1
        self._publish([row])

    def release(self, rows):
        """The rows' pages go back to the pool (those that another row shares when it
        gives them back too)."""
        self._owned()
        rows = [self._row(r) for r in (rows if isinstance(rows, (list, tuple)) else [rows])]
        if len(set(rows)) != len(rows):
            raise ValueError("Each cache row once")
        for row in rows:
            self._drop(self._held[row])
            self._held[row] = []
        if rows:
            self._publish(rows)

    def evict(self, weights, used, keep, recent=0, room=0):
        """Hold every row to ``keep`` positions (:func:`kv_paged.evict`): per layer and
        KV head the ``recent`` last and the heaviest others of the row's ``used[b]`` (no
        more than it has pages for) stay, in their order, in fresh pages; the old ones go
        back to the pool. A row that has pages for ``keep`` positions or fewer loses
        nothing: its pages stay, shared ones too, and are not copied. ``weights [L, B, H,
        capacity]`` (fp32) is compacted in place. ``room``: positions that each of the
        others gets pages for beyond ``keep``. Returns the positions kept ``[L, B, H,
        keep]`` and the rows' new ``used``; a row goes on at that position, with rotary
        positions counted from where it was."""
        self._owned()
        keep, room = int(keep), int(room)
        if room < 0 or keep + room > self.capacity:
            raise ValueError("Positions of a row exceed the KV capacity")
        moved = [row for row, pages in enumerate(self._held) if len(pages) * self.page > keep]
        each = max(0, -(-(keep + room) // self.page))
        if len(moved) * each > len(self._free):
            raise ValueError(f"The KV pool has {len(self._free)} free pages, {len(moved) * each} are wanted")
        fresh = {row: self._take(each) for row in moved}
        width = max(1, each)
        # each row's pages to come (none where it keeps its own), and the positions that it has pages for
        lines = []
        for row, old in enumerate(self._held):
            pages = fresh.get(row, [])
            lines.append(pages + [-1] * (width - len(pages)) + [len(old) * self.page])
        try:
            lines = torch.tensor(lines, dtype=torch.int32).to(self._table.device)
            used = kv_quant.per_row(used, len(self._held), torch.int32, lines.get_device(), "used")
            _, kept, left = kv_paged.evict(self, weights, used.minimum(lines[:, width]), keep, recent,
                                           lines[:, :width].contiguous(), weights_out=weights)
        except Exception:
            for pages in fresh.values():
                self._drop(pages)
            raise
        for row in moved:
            self._drop(self._held[row])
            self._held[row] = fresh[row]
        if moved:
            self._publish(moved)
        return kept, left

    # -- contents --------------------------------------------------------------
    def reset(self):
        """Zeros everywhere; rows keep their pages."""
        self._k.zero_()
        self._v.zero_()

    def clear(self, row, start, stop):
        """Positions ``start .. stop-1`` of cache row ``row`` of every layer: zeros,
        where they have pages."""
        start, stop, _ = slice(start, stop).indices(self.capacity)
        self.check_own(row, start, stop)
        positions = self.keys[start:stop]
        n = positions.numel()
        zeros = self._k.new_zeros((n, self._k.shape[2], 1, self._k.shape[4]))
        slots = torch.full((n,), self._row(row), dtype=torch.int64, device=self._k.device)
        for layer in range(self._k.shape[0]) if n else ():
            self.write(layer, zeros, zeros, positions, None, slots)

    def prefill(self, layer, slot, k, v, valid):
        """:meth:`KVCache.prefill`, into the rows' pages."""
        from .packed import PackedPrefill
        if isinstance(slot, PackedPrefill):
            self.write(layer, k[0].transpose(0, 1).unsqueeze(2), v[0].transpose(0, 1).unsqueeze(2), slot.positions,
                       None, slot.slots)
            return k, v, None
        b, h, s, d = k.shape
        rows = self.slots[slot if isinstance(slot, slice) else slice(slot, slot + 1)]
        if s > self.capacity:
            raise ValueError("Prompt width exceeds the KV capacity")
        if rows.numel() != b:
            raise ValueError("Prefill slots must name one cache row per batch row")
        for row in range(*slot.indices(self.slots.numel())) if isinstance(slot, slice) else (slot,):
            self.check_own(row, 0, s)
        zero, keep = torch.zeros((), dtype=k.dtype, device=k.device), valid[:, None, :, None]
        pos = self.keys[:s]
        flat = [torch.where(keep, x, zero).transpose(1, 2).reshape(b * s, h, 1, d) for x in (k, v)]
        self.write(layer, *flat, pos.repeat(b), None, rows.repeat_interleave(s))
        mask = (pos[:, None] >= pos[None, :])[None, None] & valid[:, None, None, :]
        return k, v, torch.where(valid[:, None, :, None], mask, (pos == 0)[None, None, None, :])

    def decode(self, layer, k, v, lengths, active):
        """:meth:`KVCache.decode`, the layer's rows laid out one after the other."""
        pos = torch.where(active, lengths, 0)
        self.write(layer, k, v, pos, active)
        mask = self.keys[None, :] < (lengths + 1)[:, None]
        mask = torch.where(active[:, None], mask, self.keys[None, :] == 0)
        return *self.read(layer), mask[:, None, None, :]

    def write(self, layer, k, v, pos, active, slots=None):
        """Masked store of ``k, v [rows, H, 1, D]`` at ``(slots, h, pos)``."""
        return kv_paged.write(self, layer, k, v, pos, active, self.slots if slots is None else slots)

    def read(self, layer):
        """The whole layer as ``k, v [B, H, C, D]``, zeros where a row has no page."""
        batch, capacity = self.slots.numel(), self.capacity
        sides = kv_paged.read(self, layer, self.keys.repeat(batch), self.slots.repeat_interleave(capacity))
        return tuple(x.view(batch, capacity, x.shape[1], x.shape[3]).transpose(1, 2) for x in sides)
