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
    """Bits of one layer's buffers ``k, v [B, H, C, 8*bits]``, ``scales [B, H, C, 4]``."""
    _lib.require_cuda(k, v, scales, what="quantised KV cache")
    bits = k.shape[-1] // 8
    if k.dim() != 4 or bits not in BITS or k.shape[-1] % 8 or v.shape != k.shape or scales.shape != (*k.shape[:3], 4):
        raise ValueError("Quantised KV cache layers are k, v [B, H, C, 8*bits] and scales [B, H, C, 4], bits 4 or 8")
    if any(t.dtype != torch.uint8 or not t.is_contiguous() for t in (k, v, scales)):
        raise ValueError("Quantised KV cache layers must be contiguous uint8")
    if v.device != k.device or scales.device != k.device:
        raise ValueError("Quantised KV cache layers must share one device")
    return bits


def _index(t, rows, dtype, device, what):
    t = t if t.dtype == dtype else t.to(dtype)
    if t.numel() != rows or t.device != device:
        raise ValueError(f"{what} needs one entry per row, on the cache's device")
    return t.contiguous()


def write(cache, layer, k, v, positions, active, slots):
    """Quantise ``k[row, h, 0, :]`` into position ``positions[row]`` of
    ``slots[row]`` for active rows (same for v), as :func:`kv_write.write`
    stores them. ``k, v [rows, H, 1, 64]`` bf16 with any strides; ``active`` may
    be None (every row). Rows out of range are skipped. One row per target."""
    kc, vc, scales = cache.layer(layer)
    bits = check_layer(kc, vc, scales)
    if k.dim() != 4 or k.shape != v.shape or k.shape[1] != kc.shape[1] or k.shape[2] != 1 or k.shape[3] != 64:
        raise ValueError("KV write takes k, v [rows, H, 1, 64] of the cache's heads")
    _lib.require_cuda(k, v, what="KV write tensors")
    if k.dtype != torch.bfloat16 or v.dtype != torch.bfloat16:
        raise ValueError("The quantised KV write supports BF16")
    device, rows = kc.device, k.shape[0]
    if k.device != device or v.device != device:
        raise ValueError("KV write tensors must be on the cache's device")
    positions = _index(positions, rows, torch.int64, device, "positions")
    slots = _index(slots, rows, torch.int64, device, "slots")
    active = None if active is None else _index(active, rows, torch.bool, device, "active")
    with torch.cuda.device(device):
        _lib.call("lm_kv_quant_write", k.data_ptr(), k.stride(0), k.stride(1), k.stride(3), v.data_ptr(),
                  v.stride(0), v.stride(1), v.stride(3), kc.data_ptr(), vc.data_ptr(), scales.data_ptr(),
                  positions.data_ptr(), _lib.ptr(active), slots.data_ptr(), rows, kc.shape[1], 64, kc.shape[2],
                  kc.shape[0], bits, _lib.stream(device))


def read(cache, layer, positions, slots):
    """What the cache stands for at ``(slots[row], h, positions[row])``:
    ``k, v [rows, H, 1, 64]`` bf16, the layout :func:`write` takes. Rows out of
    range give zeros."""
    kc, vc, scales = cache.layer(layer)
    bits = check_layer(kc, vc, scales)
    device, rows = kc.device, positions.numel()
    positions = _index(positions, rows, torch.int64, device, "positions")
    slots = _index(slots, rows, torch.int64, device, "slots")
    k, v = torch.empty(2, rows, kc.shape[1], 1, 64, dtype=torch.bfloat16, device=device)
    with torch.cuda.device(device):
        _lib.call("lm_kv_quant_read", kc.data_ptr(), vc.data_ptr(), scales.data_ptr(), positions.data_ptr(),
                  slots.data_ptr(), rows, kc.shape[1], 64, kc.shape[2], kc.shape[0], bits, k.data_ptr(),
                  v.data_ptr(), _lib.stream(device))
    return k, v
