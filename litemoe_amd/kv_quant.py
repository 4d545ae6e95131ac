"""The quantising KV-cache store and the read-back (``lm_kv_quant_write``,
``lm_kv_quant_read``) for :class:`~litemoe_amd.cache.QuantKVCache`.

A key or value vector of 64 channels is held as two blocks of 32: a
power-of-two scale (one byte) and 32 elements of 4 bits (values 0 .5 1 1.5 2 3 4
6 with a sign) or 8 bits (sign, 4 exponent and 3 mantissa bits, to 448). A cache
position of one KV head then takes 68 or 132 bytes instead of bf16's 256. The
reference keeps its cache in the model's dtype (litemoe/cache.py:7-20); the
store's arguments are those of its ``kv_write.write`` (litemoe/kv_write.py:23-29).
"""
import torch

from . import _lib

BITS = (4, 8)


def check_layer(k, v, scales):
    """``(bits, device index)`` of one layer's buffers ``k, v [B, H, C, 8*bits]``,
    ``scales [B, H, C, 4]``."""
    index, shape = k.get_device(), k.shape
    if index < 0 or v.get_device() != index or scales.get_device() != index:
        _lib.require_cuda(k, v, scales, what="quantised KV cache")
        raise ValueError("Quantised KV cache layers must share one device")
    if len(shape) != 4 or shape[3] not in (32, 64) or v.shape != shape or scales.shape != (*shape[:3], 4):
        raise ValueError("Quantised KV cache layers are k, v [B, H, C, 8*bits] and scales [B, H, C, 4], bits 4 or 8")
    if not (k.dtype == v.dtype == scales.dtype == torch.uint8 and k.is_contiguous() and v.is_contiguous()
            and scales.is_contiguous()):
        raise ValueError("Quantised KV cache layers must be contiguous uint8")
    return shape[3] // 8, index


def per_row(t, rows, dtype, index, what):
    """``t``, one entry per row on device ``index``, as a contiguous tensor of ``dtype``."""
    if t.get_device() != index or t.numel() != rows:
        raise ValueError(f"{what} needs one entry per row, on the cache's device")
    if t.dtype != dtype:
        t = t.to(dtype)
    return t if t.is_contiguous() else t.contiguous()


def _device(kc):
    """The index of the cache's GPU; a cache's own buffers are what :func:`check_layer` asks for."""
    index = kc.get_device()
    if index < 0:
        _lib.require_cuda(kc, what="quantised KV cache")
    return index


def write(cache, layer, k, v, positions, active, slots):
    """Quantise ``k[row, h, 0, :]`` into position ``positions[row]`` of
    ``slots[row]`` for active rows (same for v), as :func:`kv_write.write`
    stores them. ``k, v [rows, H, 1, 64]`` bf16 with any strides; ``active`` may
    be None (every row). Rows out of range are skipped. One row per target."""
    kc, vc, scales = cache.layer(layer)
    index = _device(kc)
    batch, heads, capacity, _ = kc.shape
    shape = k.shape
    if len(shape) != 4 or shape[1:] != (heads, 1, 64) or v.shape != shape:
        raise ValueError("KV write takes k, v [rows, H, 1, 64] of the cache's heads")
    if k.dtype != torch.bfloat16 or v.dtype != torch.bfloat16:
        raise ValueError("The quantised KV write supports BF16")
    if k.get_device() != index or v.get_device() != index:
        raise ValueError("KV write tensors must be on the cache's device")
    rows = shape[0]
    positions = per_row(positions, rows, torch.int64, index, "positions")
    slots = per_row(slots, rows, torch.int64, index, "slots")
    active = None if active is None else per_row(active, rows, torch.bool, index, "active")
    ks, vs = k.stride(), v.stride()
    _lib.call_on(index, "lm_kv_quant_write", k.data_ptr(), ks[0], ks[1], ks[3], v.data_ptr(), vs[0], vs[1], vs[3],
                 kc.data_ptr(), vc.data_ptr(), scales.data_ptr(), positions.data_ptr(), _lib.ptr(active),
                 slots.data_ptr(), rows, heads, 64, capacity, batch, cache.bits)


def read(cache, layer, positions, slots):
    """What the cache stands for at ``(slots[row], h, positions[row])``:
    ``k, v [rows, H, 1, 64]`` bf16, the layout :func:`write` takes. Rows out of
    range give zeros."""
    kc, vc, scales = cache.layer(layer)
    index = _device(kc)
    batch, heads, capacity, _ = kc.shape
    rows = positions.numel()
    positions = per_row(positions, rows, torch.int64, index, "positions")
    slots = per_row(slots, rows, torch.int64, index, "slots")
    k = torch.empty((rows, heads, 1, 64), dtype=torch.bfloat16, device=kc.device)
    v = torch.empty_like(k)
    _lib.call_on(index, "lm_kv_quant_read", kc.data_ptr(), vc.data_ptr(), scales.data_ptr(), positions.data_ptr(),
                 slots.data_ptr(), rows, heads, 64, capacity, batch, cache.bits, k.data_ptr(), v.data_ptr())
    return k, v
