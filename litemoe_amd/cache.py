"""Contiguous rank-local KV cache ``[L, B, Hkv, C, D]`` (litemoe/cache.py:7-55).

The layout is the reference's: row b of the batch owns cache page b, a whole
``capacity``-long sequence per KV head. Writes go through the masked gfx950
store (one writer per row, head and channel).

:class:`QuantKVCache` has the same interface over a cache of 4 or 8 bits per
element (:mod:`litemoe_amd.kv_quant`)."""
from typing import NamedTuple

import torch

from . import kv_quant, kv_write


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
