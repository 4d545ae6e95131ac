"""Rotary embedding, alone or fused with the KV-cache store.

``rotary_embedding`` keeps the signature of vLLM's
``_custom_ops.rotary_embedding(positions, query, key, head_size, cos_sin_cache,
is_neox)`` as the reference calls it (litemoe/model.py:58,63-64): in place on
strided ``[T, heads, D]`` views. Arithmetic matches the torch path
``q * cos + rotate_half(q) * sin`` in bf16 (model.py:66-67) bit for bit.

The reference turns whole heads in halves by a bf16 table. :func:`rotary_embedding`
and :func:`rotate_kv_write` also turn interleaved pairs, the first channels of a head
alone, and by an fp32 table (:func:`rotary_table`), whose products and sums stay fp32
and are rounded once: a bf16 cosine is off by 2^-9, whatever the position.
"""
import math

import torch

from . import _lib, kv_paged
from .cache import PagedKVCache
from .kv_quant import per_row


def rotary_table(length, rotary, theta, scaling=None, device="cpu", dtype=torch.float32):
    """cos | sin ``[length, rotary]`` of positions ``0 .. length-1``, angles formed in
    64 bits. ``scaling``, for contexts ``factor`` times longer than the ``original``
    positions that the frequencies were made for:

    * ``dict(type="linear", factor=)``: every frequency divided by it;
    * ``dict(type="ntk", factor=)``: ``theta`` times ``factor ** (rotary / (rotary - 2))``,
      which divides the lowest frequency by it and leaves the highest;
    * ``dict(type="yarn", factor=, original=)`` (Peng et al., 2023): pairs that turn more
      than ``beta_fast`` (32) times within ``original`` positions keep their frequency,
      those that turn less than ``beta_slow`` (1) times have it divided, with a ramp
      between, and the values are times ``attention_factor`` (``0.1 ln(factor) + 1``)."""
    if length < 1 or rotary < 2 or rotary % 2 or theta <= 0:
        raise ValueError("A rotary table needs positions and an even number of channels")
    scaling = dict(scaling or {})
    kind, factor = scaling.pop("type", None), float(scaling.pop("factor", 1.0))
    allowed = {None: set(), "linear": set(), "ntk": set(),
               "yarn": {"original", "beta_fast", "beta_slow", "attention_factor"}}
    if kind not in allowed or factor < 1 or set(scaling) - allowed[kind] or (kind is None and factor != 1):
        raise ValueError("Rotary scaling is linear, ntk or yarn, with a factor of at least 1")
    if kind == "ntk":
        if rotary < 4:
            raise ValueError("Rotary scaling by the base needs two pairs")
        theta = theta * factor ** (rotary / (rotary - 2))
    i = torch.arange(rotary // 2, dtype=torch.float64, device=device)
    frequency, size = theta ** (-2 * i / rotary), 1.0
    if kind == "linear":
        frequency = frequency / factor
    elif kind == "yarn":
        if "original" not in scaling:
            raise ValueError("YaRN scaling needs the original positions")

        def pair(turns):  # the index of the pair that turns so often within the original positions
            return rotary * math.log(scaling["original"] / (turns * 2 * math.pi)) / (2 * math.log(theta))
        low = max(math.floor(pair(scaling.get("beta_fast", 32.0))), 0)
        high = min(math.ceil(pair(scaling.get("beta_slow", 1.0))), rotary - 1)
        ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
        frequency = frequency * (1 - ramp) + frequency / factor * ramp
        size = scaling.get("attention_factor")
        size = 0.1 * math.log(factor) + 1 if size is None else size
    angle = torch.arange(length, dtype=torch.float64, device=device)[:, None] * frequency
    return (torch.cat((angle.cos(), angle.sin()), -1) * size).to(dtype)


def check_table(cos_sin, index, dim):
    """``cos_sin [table_len, rotary]`` as the kernels with any rotation take it."""
    shape = cos_sin.shape
    if (cos_sin.dtype not in (torch.float32, torch.bfloat16) or len(shape) != 2 or not cos_sin.is_contiguous()
            or cos_sin.get_device() != index or not shape[0] or cos_sin.data_ptr() % 16):
        raise ValueError("Rotation needs a contiguous FP32 or BF16 [table_len, rotary] cos/sin table on one device "
                         "with its tensors")
    if shape[1] % 16 or not 16 <= shape[1] <= dim:
        raise ValueError("Rotated channels are a multiple of 16, at most the head's")


SHARED = "Rotation in place needs queries and keys whose rows and heads share no memory"


def _check(q, k, cos_sin, positions):
    _lib.require_cuda(q, k, cos_sin, positions, what="RoPE tensors")
    if q.dtype != torch.bfloat16 or k.dtype != torch.bfloat16 or cos_sin.dtype != torch.bfloat16:
        raise ValueError('RoPE supports BF16 query/key/table')
    if q.stride(-1) != 1 or k.stride(-1) != 1 or not cos_sin.is_contiguous():
        raise ValueError('RoPE needs contiguous channels and a contiguous cos/sin table')
    if q.shape[-1] != 64 or k.shape[-1] != 64 or cos_sin.shape[-1] != 64:
        raise ValueError('RoPE kernel supports head_dim 64')
    for t in (q, k):
        if t.stride(0) % 8 or t.stride(1) % 8 or t.data_ptr() % 16:
            raise ValueError('RoPE needs 16-byte aligned rows and heads (strides multiple of 8)')


def _apart(q, k):
    """Whether every head of ``q`` and of ``k`` (``[T, heads, D]``, contiguous channels) has memory of its own, as a
    rotation in place needs it."""
    (rows, heads, *_, dim), (s0, s1, *_) = q.shape, q.stride()
    (k_rows, k_heads, *_, k_dim), (k0, k1, *_) = k.shape, k.stride()
    width, k_width = (heads - 1) * s1 + dim, (k_heads - 1) * k1 + k_dim  # of a row
    at = (k.data_ptr() - q.data_ptr()) // 2
    rows_apart = (s0 >= width or rows == 1) and (k0 >= k_width or k_rows == 1)
    if rows_apart and (s1 >= dim or heads == 1) and (k1 >= k_dim or k_heads == 1):
        if at >= (rows - 1) * s0 + width or -at >= (k_rows - 1) * k0 + k_width:
            return True  # one behind the other
        if 0 < s0 == k0 and width <= at % s0 <= s0 - k_width:
            return True  # columns of the same rows
    if not q.numel():
        rows, heads, width = 0, 0, 0
    if not k.numel():
        k_rows, k_heads, k_width = 0, 0, 0
    if (heads <= 1 or s1 >= (rows - 1) * s0 + dim) and (k_heads <= 1 or k1 >= (k_rows - 1) * k0 + k_dim) \
            and (rows <= 1 or s0 >= dim) and (k_rows <= 1 or k0 >= k_dim):
        # of each head all rows, then the next head's
        if at >= (heads - 1) * s1 + (rows - 1) * s0 + dim or -at >= (k_heads - 1) * k1 + (k_rows - 1) * k0 + k_dim:
            return True

    def free(starts, ends):
        starts, order = starts.sort()
        return not bool((starts[1:] < ends[order][:-1]).any())

    def all_of(rows, heads, step, inner, dim, base):
        starts = (base + step * torch.arange(rows, device="cpu")[:, None]
                  + inner * torch.arange(heads, device="cpu")).flatten()
        return starts, starts + dim
    if rows_apart and s0 == k0 > 0 and min(rows, k_rows) > 1:
        # rows repeat: the heads of one row, of what reaches into the next its place there too
        of_row = zip(all_of(1, heads, 0, s1, dim, 0), all_of(1, k_heads, 0, k1, k_dim, at % s0))
        if free(*(torch.cat((x, y, x + s0, y + s0)) for x, y in of_row)):
            return True
    whole = zip(all_of(rows, heads, s0, s1, dim, 0), all_of(k_rows, k_heads, k0, k1, k_dim, at))
    return free(*(torch.cat(x) for x in whole))


def rotary_embedding(positions, query, key, head_size, cos_sin_cache, is_neox=True):
    """In-place rotation of ``query [T, Hq, D]`` and ``key [T, Hkv, D]`` by the table
    ``cos_sin_cache [table_len, R]``: its width says how many of a head's channels
    turn, and its type the arithmetic (see :func:`rotate_kv_write`). ``is_neox``: pairs
    in halves, else interleaved. Rows and heads have memory of their own, within each
    tensor and between the two."""
    if head_size != query.shape[-1]:
        raise ValueError('head_size must equal the last query dimension')
    if is_neox and head_size == 64 and cos_sin_cache.shape[-1] == 64 and cos_sin_cache.dtype == torch.bfloat16:
        _check(query, key, cos_sin_cache, positions)
        if not _apart(query, key):
            raise ValueError(SHARED)
        positions = positions.to(torch.int64).contiguous()
        rows = query.shape[0]
        _lib.call("lm_rope_kv_write", query.data_ptr(), query.stride(0), query.stride(1),
                  key.data_ptr(), key.stride(0), key.stride(1), None, 0, 0,
                  cos_sin_cache.data_ptr(), cos_sin_cache.shape[0], positions.data_ptr(), None, None,
                  None, None, rows, query.shape[1], key.shape[1], 64, 1, 1, 1, _lib.stream(query.device))
        return
    for t in (query, key):
        if t.dim() != 3 or t.dtype != torch.bfloat16 or kv_paged.view(t, *t.shape[:2])[0] is not t:
            raise ValueError('Rotation in place needs BF16 [T, heads, D] of contiguous channels, 16-byte aligned rows '
                             'and heads (strides multiple of 8)')
    if not _apart(query, key):
        raise ValueError(SHARED)
    _rotate(query, key, positions, cos_sin_cache, is_neox, query, key)


def _rotate(q, k, positions, cos_sin, is_neox, q_out, k_out, v=None, cache=None, layer=0, at=None, active=None,
            slots=None):
    """The call of ``lm_paged_rotate_write`` on BF16 ``[T, heads, D]``; the rest is checked.
    Results go to ``q_out`` and ``k_out``, new and contiguous or the operands themselves."""
    rows, q_heads, dim = q.shape
    k_rows, k_heads, k_dim = k.shape
    index = q.get_device()
    if index < 0:
        _lib.require_cuda(q, k, cos_sin, what="RoPE tensors")
    if k_rows != rows or k_dim != dim or k.get_device() != index:
        raise ValueError("Queries and keys need the same rows and channels, on one device")
    if dim % 16 or dim > 256:
        raise ValueError("Rotation takes heads of a multiple of 16 channels, at most 256")
    check_table(cos_sin, index, dim)
    positions = per_row(positions, rows, torch.int64, index, "positions")
    q_in, q_view = kv_paged.view(q, rows, q_heads)
    k_in, k_view = kv_paged.view(k, rows, k_heads)
    where, v_view, place, i32, slot, mask = (0,) * 7, (0, 0, 0), 0, False, 0, 0
    if cache is not None:
        kc, vc, table = cache.layer(layer)
        if kv_paged.check_layer(kc, vc, table) != index:
            raise ValueError("The cache must be on its tensors' device")
        pages, heads, page, channels = kc.shape
        if heads != k_heads or channels != dim or v.shape != k.shape or v.get_device() != index:
            raise ValueError("Keys and values do not match the cache's heads")
        v_in, v_view = kv_paged.view(v, rows, heads)
        if at is not None:
            at = kv_paged.places(at, rows, index, "at")
            place, i32 = at.data_ptr(), at.dtype is torch.int32
        if slots is not None:
            slots = per_row(slots, rows, torch.int64, index, "slots")
            slot = slots.data_ptr()
        if active is not None:
            active = per_row(active, rows, torch.bool, index, "active")
            mask = active.data_ptr()
        where = kc.data_ptr(), vc.data_ptr(), table.data_ptr(), *table.shape, pages, page
    q_to = q_view if q_out is q else (q_out.data_ptr(), q_heads * dim, dim)
    k_to = k_view if k_out is k else (0, 0, 0) if k_out is None else (k_out.data_ptr(), k_heads * dim, dim)
    _lib.call_struct(index, "lm_paged_rotate_write", *q_view, *k_view, *v_view, cos_sin.data_ptr(), *cos_sin.shape,
                     cos_sin.dtype is torch.float32, bool(is_neox), positions.data_ptr(), place, i32, mask, slot, *q_to,
                     *k_to, *where, rows, q_heads, k_heads, dim)


def rotate_kv_write(q, k, v, positions, active, cos_sin, cache, layer, slots=None, at=None, is_neox=True, keep_k=False):
    """Rotate ``q [T, Hq, D]`` and ``k [T, Hkv, D]`` by ``positions``, and store rotated k
    and ``v`` into a :class:`~litemoe_amd.cache.PagedKVCache` at ``(slots[t], h, at[t])``
    for active rows (``slots`` None: row t; ``at`` None: ``positions``, which a row that
    was evicted from has moved past; ``active`` None: all). Rows out of range or without
    a page there are not stored. Returns the rotated ``q``, and with ``keep_k`` the
    rotated ``k`` (else None), as new tensors.

    The first ``R`` channels turn, for a table ``cos_sin [table_len, R]``, in halves
    (``is_neox``) or interleaved pairs; positions past the table are not turned. An
    fp32 table: fp32 arithmetic, rounded once. A bf16 table: each product and each sum
    is rounded, as :func:`rope_kv_write` and litemoe/model.py:66-67 have it."""
    if not isinstance(cache, PagedKVCache):
        raise ValueError("rotate_kv_write stores into a paged KV cache")
    for t in (q, k, v):
        if t.dtype is not torch.bfloat16 or t.dim() != 3:
            raise ValueError("RoPE supports BF16 [T, heads, D] queries, keys and values")
    q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
    k_out = torch.empty_like(k, memory_format=torch.contiguous_format) if keep_k else None
    _rotate(q, k, positions, cos_sin, is_neox, q_out, k_out, v, cache, layer, at, active, slots)
    return q_out, k_out


def rope_kv_write(q, k, v, positions, active, cos_sin, cache, layer, slots=None, write_k=False):
    """Rotate ``q`` (in place) and ``k``, store rotated k and v into ``cache`` at
    ``(slots[r], h, positions[r])`` for active rows. ``q [T, Hq, 64]``,
    ``k, v [T, Hkv, 64]`` strided views (e.g. of the packed QKV projection).
    ``write_k`` also writes rotated k back in place (prefill attends over it).
    Replaces rotary_embedding + cache.write (litemoe/model.py:58-59, :64-70)."""
    _check(q, k, cos_sin, positions)
    kc, vc = cache.k[layer], cache.v[layer]
    if v.stride(-1) != 1 or v.dtype != torch.bfloat16 or kc.dtype != torch.bfloat16:
        raise ValueError('Fused RoPE/KV write needs BF16 v and cache with contiguous channels')
    if v.stride(0) % 8 or v.stride(1) % 8 or v.data_ptr() % 16:
        raise ValueError('RoPE needs 16-byte aligned v rows and heads (strides multiple of 8)')
    rows = q.shape[0]
    positions = positions.to(torch.int64).contiguous()
    active = active.to(torch.bool).contiguous()
    slots = None if slots is None else slots.to(torch.int64).contiguous()
    _lib.call("lm_rope_kv_write", q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(),
              k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), cos_sin.data_ptr(),
              cos_sin.shape[0], positions.data_ptr(), active.data_ptr(), _lib.ptr(slots),
              kc.data_ptr(), vc.data_ptr(), rows, q.shape[1], k.shape[1], 64, cache.capacity,
              kc.shape[0], int(bool(write_k)), _lib.stream(q.device))
