"""The paged KV cache without a GPU: pages handed out and given back, tables, rotary
tables, and the calls that are refused before anything is launched."""
import copy
import math
import pickle
import re
import weakref
from pathlib import Path

import pytest
import torch

from litemoe_amd import _lib, kv_paged, kv_quant, rope
from litemoe_amd.cache import KVCache, PagedKVCache
from litemoe_amd.config import preset
from litemoe_amd.engine import Engine
from litemoe_amd.flash_decode import PagedFlashDecode, paged_shares, paged_splits
from oracle import paged

_P = 1 << 20


def cache_of(rows=3, capacity=64, page=16, pages=None):
    return PagedKVCache.empty(2, rows, 4, 64, capacity, "cpu", page=page, pages=pages)


def lines(cache):
    return [[p for p in line if p >= 0] for line in cache.table.tolist()]


def test_sizes():
    cfg = preset("granite-3b", num_hidden_layers=2)
    cache = PagedKVCache(cfg, 3, 100, "cpu", torch.bfloat16, page=32, pages=7)
    assert cache.k.shape == cache.v.shape == (2, 7, 8, 32, 64)
    assert cache.table.shape == (3, 4) and cache.capacity == 128 and cache.page == 32
    assert cache.slots.tolist() == [0, 1, 2] and cache.keys.numel() == 128
    assert bool((cache.table == -1).all()) and cache.free_pages == 7
    layer = cache.layer(1)
    assert layer.k.data_ptr() == cache.k[1].data_ptr() and layer.table is cache.table
    assert PagedKVCache(cfg, 3, 100, "cpu", torch.bfloat16).k.shape[1] == 6


def test_pages_are_handed_out_and_given_back():
    cache = cache_of(pages=8)
    cache.reserve([0, 1], [17, 16])
    assert [len(x) for x in lines(cache)] == [2, 1, 0] and cache.free_pages == 5
    assert cache.held(0) == 32 and cache.held(2) == 0
    first = lines(cache)
    cache.reserve([0, 1], [17, 20])  # what a row has stays in its place
    assert lines(cache)[0] == first[0] and lines(cache)[1][:1] == first[1] and len(lines(cache)[1]) == 2
    used = [p for line in lines(cache) for p in line]
    assert len(set(used)) == len(used)
    before = cache.table.clone()
    with pytest.raises(ValueError, match="4 free pages, 6 are wanted"):
        cache.reserve([0, 2], [64, 64])
    assert torch.equal(cache.table, before) and cache.free_pages == 4
    cache.release(0)
    assert lines(cache)[0] == [] and cache.free_pages == 6 and cache.held(0) == 0
    cache.reserve(2, 64)
    assert len(lines(cache)[2]) == 4
    cache.release([1, 2])
    assert cache.free_pages == 8 and bool((cache.table == -1).all())


def test_shared_pages_go_back_when_the_last_row_gives_them_back():
    cache = cache_of(pages=6)
    cache.reserve(0, 40)
    cache.share(1, 0, 32)
    assert lines(cache)[1] == lines(cache)[0][:2] and cache.free_pages == 3
    cache.reserve(1, 48)
    assert len(set(lines(cache)[0] + lines(cache)[1])) == 4
    cache.release(0)
    assert cache.free_pages == 3
    cache.release(1)
    assert cache.free_pages == 6
    for args, text in [((0, 0, 0), "without pages"), ((0, 1, 16), "whole pages"), ((0, 5, 0), "No such")]:
        with pytest.raises(ValueError, match=text):
            cache.share(*args)
    cache.reserve([0, 1], 16)
    with pytest.raises(ValueError, match="without pages"):
        cache.share(0, 1, 16)
    with pytest.raises(ValueError, match="whole pages"):
        cache.share(2, 1, 8)


@pytest.mark.parametrize("call,text", [
    (lambda c: c.reserve(3, 16), "No such"), (lambda c: c.reserve(-1, 16), "No such"),
    (lambda c: c.reserve(0, 65), "capacity"), (lambda c: c.reserve(0, -1), "capacity"),
    (lambda c: c.reserve([0, 0], 16), "once"), (lambda c: c.reserve([0, 1], [16]), "capacity"),
    (lambda c: c.release([1, 1]), "once"), (lambda c: c.release(9), "No such"),
    (lambda c: c.evict(None, None, 60, room=10), "capacity"), (lambda c: c.evict(None, None, 4, room=-1), "capacity"),
])
def test_page_calls_refused(call, text):
    cache = cache_of()
    cache.reserve([0, 1], 20)
    before = cache.table.clone()
    with pytest.raises(ValueError, match=text):
        call(cache)
    assert torch.equal(cache.table, before) and cache.free_pages == 8


def test_a_refused_eviction_gives_its_pages_back():
    cache = cache_of()
    cache.reserve([0, 1], 40)
    before, free = cache.table.clone(), cache.free_pages
    weights = torch.zeros(2, 3, 4, 64)
    with pytest.raises(ValueError, match="ROCm device"):
        cache.evict(weights, torch.tensor([40, 40, 0]), 16)
    assert torch.equal(cache.table, before) and cache.free_pages == free
    tight = cache_of(pages=6)
    tight.reserve([0, 1], 40)
    with pytest.raises(ValueError, match="0 free pages, 2 are wanted"):
        tight.evict(weights, torch.tensor([40, 40, 0]), 16)


def test_an_eviction_leaves_rows_that_lose_nothing(monkeypatch):
    """Rows with pages for no more than the budget keep them, in a pool that has free pages for the others only; a
    shared beginning stays shared."""
    cache = cache_of(rows=4, pages=10)
    cache.reserve([0, 1], [64, 32])
    cache.share(2, 1, 32)
    cache.reserve(2, 48)
    before, targets = lines(cache), []
    assert cache.free_pages == 3

    def moved(cache, weights, used, keep, recent, target, table=None, weights_out=None):
        targets.append([[p for p in line if p >= 0] for line in target.tolist()])
        return weights_out, None, used.clamp(max=keep)
    monkeypatch.setattr(kv_paged, "evict", moved)
    weights = torch.zeros(2, 4, 4, 64)
    _, left = cache.evict(weights, torch.tensor([60, 40, 48, 5]), 48)
    assert left.tolist() == [48, 32, 48, 0]
    assert len(targets[0][0]) == 3 and targets[0][1:] == [[], [], []]
    assert lines(cache) == [targets[0][0], *before[1:]] and lines(cache)[2][:2] == lines(cache)[1]
    assert cache.free_pages == 10 - 3 - 3 and not set(lines(cache)[0]) & set(lines(cache)[2])
    # nothing to evict: no free page is asked for
    cache.reserve([1, 3], [64, 32])
    assert cache.free_pages == 0
    full = lines(cache)
    cache.evict(weights, torch.tensor([48, 64, 48, 32]), 64)
    assert lines(cache) == full and targets[1] == [[]] * 4
    cache.release([0, 1, 2, 3])
    assert cache.free_pages == 10


def test_stores_by_rows_keep_out_of_shared_pages(monkeypatch):
    """After ``share`` neither row's first pages are cleared or prefilled; what lies behind them is, and all of it
    when one of the rows has given them back."""
    cache = cache_of(rows=3, pages=12)
    cache.reserve([0, 2], 64)
    cache.share(1, 0, 32)
    cache.reserve(1, 64)
    stored = []
    monkeypatch.setattr(kv_paged, "write", lambda cache, layer, k, v, at, active, slots: stored.append(
        sorted(set(zip(slots.tolist(), at.tolist())))))

    def prefill(slot, width, rows=1):
        x = torch.zeros(rows, 4, width, 64, dtype=torch.bfloat16)
        return cache.prefill(0, slot, x, x, torch.ones(rows, width, dtype=torch.bool))
    for call in (lambda: cache.clear(1, 0, 8), lambda: cache.clear(0, 31, 40), lambda: cache.clear(1, -64, 20),
                 lambda: prefill(1, 1), lambda: prefill(0, 64), lambda: prefill(slice(1, 3), 20, 2),
                 lambda: prefill(slice(0, 3), 3, 3)):
        with pytest.raises(ValueError, match="shares"):
            call()
    assert not stored
    cache.clear(1, 32, 40)
    cache.clear(0, 20, 20)
    cache.clear(2, 0, 3)
    assert stored == 2 * [[(1, j) for j in range(32, 40)]] + 2 * [[(2, j) for j in range(3)]]
    prefill(2, 5)
    cache.release(0)
    prefill(slice(0, 3), 2, 3)
    assert stored[-2:] == [[(2, j) for j in range(5)], [(i, j) for i in range(3) for j in range(2)]]
    # pages that are the caller's to hand out are not looked at
    other = PagedKVCache.over(cache.k, cache.v, torch.zeros(3, 4, dtype=torch.int32))
    other.clear(1, 0, 4)


def test_a_cache_over_buffers():
    k = torch.zeros(2, 5, 4, 16, 64, dtype=torch.bfloat16)
    table = torch.zeros(3, 2, dtype=torch.int32)
    cache = PagedKVCache.over(k, k.clone(), table)
    assert cache.k is k and cache.table is table and cache.capacity == 32
    for call in (lambda: cache.reserve(0, 1), lambda: cache.release(0), lambda: cache.share(0, 1, 0),
                 lambda: cache.free_pages, lambda: cache.held(0), lambda: cache.evict(None, None, 1)):
        with pytest.raises(ValueError, match="caller's"):
            call()
    for args, text in [((k[0], k[0], table), "buffers are"), ((k, k[:, :, :2], table), "buffers are"),
                       ((k[..., :32].contiguous(), k[..., :32].contiguous(), table), "buffers are"),
                       ((k[:, :, :, :8].contiguous(), k[:, :, :, :8].contiguous(), table), "buffers are"),
                       ((k.float(), k.float(), table), "BF16"), ((k[:, 1:], k[:, 1:], table), "contiguous"),
                       ((k, k, table.long()), "int32"), ((k, k, table[:, :1]), "int32"), ((k, k, table[0]), "int32")]:
        with pytest.raises(ValueError, match=text):
            PagedKVCache.over(*args)


@pytest.mark.parametrize("twin", [copy.deepcopy, lambda c: pickle.loads(pickle.dumps(c))])
def test_a_copy_has_buffers_and_pages_of_its_own(twin):
    cache = cache_of()
    cache.reserve(0, 20)
    other = twin(cache)
    other.reserve(1, 16)
    other.layer(1).k.fill_(3)
    assert bool((other.k[1] == 3).all()) and not cache.k.any()
    assert other.layer(0).table.data_ptr() == other.table.data_ptr() and lines(cache)[1] == []
    assert cache.free_pages == other.free_pages + 1


@pytest.mark.parametrize("kwargs,text", [
    (dict(page=24), "power of two"), (dict(page=8), "power of two"), (dict(page=1 << 17), "power of two"),
    (dict(pages=0), "needs"), (dict(dtype=torch.float32), "BF16"), (dict(batch=0), "needs"),
])
def test_caches_refused(kwargs, text):
    cfg = preset("granite-1b", num_hidden_layers=1)
    args = dict(cfg=cfg, batch=2, capacity=64, device="cpu", dtype=torch.bfloat16, **{})
    with pytest.raises(ValueError, match=text):
        PagedKVCache(**{**args, **kwargs})
    if "page" in kwargs:
        with pytest.raises(ValueError, match="power of two"):
            Engine(None, [], kv_page=kwargs["page"])
    with pytest.raises(ValueError, match="16 bits"):
        Engine(None, [], kv_page=16, kv_bits=8)


def test_host_tensors_are_refused():
    cache = cache_of()
    x, at = torch.zeros(3, 4, 1, 64, dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int64)
    flash = PagedFlashDecode(3, 4, 2, cache.capacity, "cpu")
    cos_sin = rope.rotary_table(16, 64, 1e4)
    q = torch.zeros(3, 8, 1, 64, dtype=torch.bfloat16)
    for call in (lambda: cache.write(0, x, x, at, None), lambda: cache.read(0),
                 lambda: flash(q, *cache.layer(0), None, None, 1.0, used=at),
                 lambda: flash.fused_qkv(torch.zeros(1, 3, 16 * 64), cos_sin, at, None, *cache.layer(0), 1.0, at, 8),
                 lambda: rope.rotate_kv_write(q[:, :, 0], x[:, :, 0], x[:, :, 0], at, None, cos_sin, cache, 0),
                 lambda: rope.rotary_embedding(at, q[:, :, 0], x[:, :, 0], 64, cos_sin, is_neox=False),
                 lambda: kv_paged.evict(cache, torch.zeros(2, 3, 4, 64), at, 2, 0, cache.table)):
        with pytest.raises(ValueError, match="ROCm device"):
            call()
    plain = KVCache(preset("granite-1b", num_hidden_layers=1), 1, 16, "cpu", torch.bfloat16)
    with pytest.raises(ValueError, match="paged KV cache"):
        rope.rotate_kv_write(q[:, :, 0], x[:, :, 0], x[:, :, 0], at, None, cos_sin, plain, 0)


@pytest.mark.parametrize("call", ["write", "read", "rotate", "attend", "fused"])
def test_converted_arguments_live_through_the_call(call, monkeypatch):
    """What a call converts or copies (a mask of bytes, places of another type, operands without alignment) is held
    until its kernel is launched: memory given back before is the next copy's."""
    made, missing = [], []

    def recorded(function, result):
        def wrapper(*args, **kwargs):
            out = function(*args, **kwargs)
            made.append(weakref.ref(result(out)))
            return out
        return wrapper
    monkeypatch.setattr(kv_quant, "per_row", recorded(kv_quant.per_row, lambda t: t))
    for module in (kv_paged, rope):
        monkeypatch.setattr(module, "per_row", kv_quant.per_row)
    monkeypatch.setattr(kv_paged, "view", recorded(kv_paged.view, lambda out: out[0]))
    # the calls as far as their launch, on host tensors
    monkeypatch.setattr(kv_paged, "check_layer", lambda k, v, table: -1)
    monkeypatch.setattr(_lib, "require_cuda", lambda *tensors, what: None)
    monkeypatch.setattr(_lib, "call_struct", lambda *args: missing.extend(r for r in made if r() is None))
    cache = cache_of()
    odd = torch.zeros(3, 4, 1, 65, dtype=torch.bfloat16)[..., 1:]
    q, cos_sin = torch.zeros(3, 8, 1, 65, dtype=torch.bfloat16)[..., 1:], rope.rotary_table(16, 64, 1e4)
    at, mask, short = torch.zeros(6, dtype=torch.int16)[::2], torch.ones(3, dtype=torch.uint8), torch.ones(3).short()
    flash = PagedFlashDecode(3, 4, 2, cache.capacity, "cpu")
    if call == "write":
        cache.write(0, odd, odd, at, mask, short)
    elif call == "read":
        kv_paged.read(cache, 0, at, short)
    elif call == "rotate":
        rope.rotate_kv_write(q[:, :, 0], odd[:, :, 0], odd[:, :, 0], short, mask, cos_sin, cache, 0, short, at=at)
    elif call == "attend":
        flash(torch.zeros(3, 8, 1, 64, dtype=torch.bfloat16), *cache.layer(0), None, None, 1.0, used=short)
    else:
        flash.fused_qkv(torch.zeros(1, 3, 16 * 64), cos_sin, short, mask, *cache.layer(0), 1.0, short, 8)
    assert made and not missing


def heads_of(x, rows, heads, dim, s0, s1, offset=0):
    """``[rows, heads, dim]`` within the buffer ``x``."""
    return x.as_strided((rows, heads, dim), (s0, s1, 1), offset)


# q's and k's rows, heads, strides and offset in one buffer
APART = [
    ((4, 4, 256, 64, 0), (4, 2, 128, 64, 1024)),            # one behind the other
    ((4, 4, 512, 64, 0), (4, 2, 512, 64, 256)),             # columns of one projection
    ((4, 2, 512, 64, 256), (4, 4, 512, 64, 384)),           # k's columns behind, q's first ones missing
    ((4, 4, 512, 64, 128), (4, 2, 512, 64, 0)),             # k's columns before q's
    ((4, 3, 576, 192, 0), (4, 3, 576, 192, 64)),            # heads in turn: q, k, v of each
    ((1, 3, 0, 192, 0), (1, 3, 0, 192, 64)),                # of a single row
    ((4, 4, 64, 256, 0), (4, 2, 64, 256, 1024)),            # heads outside, rows inside
    ((2, 2, 128, 192, 0), (1, 1, 0, 0, 64)),                # neither nested in the other
    ((3, 1, 128, 0, 0), (3, 1, 128, 0, 64)),                # rows in turn
    ((0, 4, 256, 64, 0), (0, 4, 256, 64, 0)),               # no rows
]
OVERLAP = [
    ((4, 4, 128, 32, 0), (4, 2, 128, 64, 2048)),            # heads half over the next
    ((4, 4, 192, 64, 0), (4, 2, 128, 64, 2048)),            # rows over the next row's first head
    ((4, 2, 256, 64, 2048), (4, 4, 32, 256, 0)),            # k's rows
    ((4, 4, 256, 64, 0), (4, 4, 256, 64, 0)),               # one tensor as both
    ((4, 4, 512, 64, 0), (4, 2, 512, 64, 192)),             # k begins in q's last head
    ((4, 2, 512, 64, 448), (4, 2, 512, 64, 0)),             # q's last head is the next row's first of k
    ((4, 3, 576, 192, 0), (4, 3, 576, 192, 32)),            # heads in turn, half over each other
    ((1, 1, 0, 0, 32), (1, 3, 0, 64, 0)),
    ((2, 2, 128, 192, 0), (1, 1, 0, 0, 96)),
    ((4, 1, 0, 0, 0), (4, 1, 64, 0, 1024)),                 # one row for all
]


@pytest.mark.parametrize("whole", [False, True])
@pytest.mark.parametrize("q,k,fine", [(*x, True) for x in APART] + [(*x, False) for x in OVERLAP])
def test_rotation_in_place_needs_memory_of_its_own(q, k, fine, whole, monkeypatch):
    """Heads that share memory, a tensor's own or those of queries and keys, would be turned by threads at once, some
    of them twice: refused before the launch, by either kernel (``whole``: the reference's bf16 table)."""
    def shares(*views):
        seen = set()
        for rows, heads, s0, s1, offset in views:
            for start in (offset + r * s0 + h * s1 for r in range(rows) for h in range(heads)):
                cells = set(range(start, start + 64))
                if seen & cells:
                    return True
                seen |= cells
        return False
    assert shares(q, k) is not fine
    launched = []
    monkeypatch.setattr(_lib, "require_cuda", lambda *tensors, what: None)
    monkeypatch.setattr(_lib, "stream", lambda device: None)
    for name in ("call", "call_struct"):
        monkeypatch.setattr(_lib, name, lambda *args: launched.append(args))
    x = torch.zeros(4096, dtype=torch.bfloat16)
    query, key = (heads_of(x, rows, heads, 64, s0, s1, offset) for rows, heads, s0, s1, offset in (q, k))
    if query.shape[0] != key.shape[0]:  # the call needs the same rows: the check itself
        assert rope._apart(query, key) is fine
        return
    cos_sin = rope.rotary_table(16, 64, 1e4, dtype=torch.bfloat16 if whole else torch.float32)
    at = torch.zeros(query.shape[0], dtype=torch.int64)
    if fine:
        rope.rotary_embedding(at, query, key, 64, cos_sin)
        assert launched
    else:
        with pytest.raises(ValueError, match="in place"):
            rope.rotary_embedding(at, query, key, 64, cos_sin)
        assert not launched


def test_rotation_in_place_of_single_positions(monkeypatch):
    """The reference's table takes ``[T, heads, 1, 64]`` too, as a decode step has its heads."""
    launched = []
    monkeypatch.setattr(_lib, "require_cuda", lambda *tensors, what: None)
    monkeypatch.setattr(_lib, "stream", lambda device: None)
    monkeypatch.setattr(_lib, "call", lambda *args: launched.append(args))
    q, k, _ = torch.zeros(5, 12, 1, 64, dtype=torch.bfloat16).split((8, 2, 2), 1)
    at, cos_sin = torch.zeros(5, dtype=torch.int64), rope.rotary_table(16, 64, 1e4, dtype=torch.bfloat16)
    rope.rotary_embedding(at, q, k, 64, cos_sin)
    assert launched[0][1:7] == (q.data_ptr(), 768, 64, k.data_ptr(), 768, 64)
    with pytest.raises(ValueError, match="in place"):
        rope.rotary_embedding(at, q, q[:, 1:], 64, cos_sin)


@pytest.mark.parametrize("kwargs,text", [(dict(maximum=0), "length bound"), (dict(maximum=65), "length bound"),
                                         (dict(head_dim=32), "head_dim"), (dict(groups=17), "16 query heads"),
                                         (dict(groups=0), "16 query heads")])
def test_plans_refused(kwargs, text):
    with pytest.raises(ValueError, match=text):
        PagedFlashDecode(**{**dict(batch=2, kv_heads=4, groups=2, capacity=64, device="cpu"), **kwargs})


def test_pieces_are_within_bounds():
    for batch in (1, 2, 3, 8, 17, 32, 33, 64, 128, 1000, 3000):
        for heads in (1, 2, 8, 32):
            for maximum in (1, 16, 255, 767, 768, 1279, 4095, 32768, 1 << 20):
                splits = paged_splits(batch, heads, maximum)
                assert 1 <= splits <= 256 and (splits == 1 or maximum >= 128 * splits)
                for dim in (64, 128):
                    assert 0 <= paged_shares(batch, heads, maximum, dim) <= 512


# ------------------------------------------------------------ rotary tables --

@pytest.mark.parametrize("rotary,theta", [(64, 10000.0), (128, 1e6), (2, 100.0)])
def test_rotary_table_is_the_definition(rotary, theta):
    """Angles in 64 bits: at position 10^6 an fp32 angle is off by up to 0.03."""
    table = rope.rotary_table(1_000_001, rotary, theta)
    at = torch.tensor([0, 1, 999, 1_000_000])
    cos, sin = paged.angles(at, rotary, theta)
    exp = torch.cat((cos, sin), -1)
    # one rounding to fp32, and an angle in 64 bits: 10^6 2^-53 and theta's power's few of its own
    assert bool(((table[at].double() - exp).abs() <= 2.0 ** -24 + 1e-8).all())
    assert table.dtype == torch.float32 and table.shape == (1_000_001, rotary)


def test_rotary_scaling():
    linear = rope.rotary_table(64, 32, 1e4, dict(type="linear", factor=4.0), dtype=torch.float64)
    plain = rope.rotary_table(16, 32, 1e4, dtype=torch.float64)
    assert torch.allclose(linear[::4], plain, atol=1e-13)
    ntk = rope.rotary_table(2, 32, 1e4, dict(type="ntk", factor=8.0), dtype=torch.float64)
    angle = torch.atan2(ntk[1, 16:], ntk[1, :16])
    base = 1e4 ** (-torch.arange(16).double() / 16)
    assert math.isclose(float(angle[0]), 1.0, rel_tol=1e-12)
    assert math.isclose(float(angle[-1]), float(base[-1]) / 8, rel_tol=1e-9)
    # YaRN: the fastest pairs as they were, the slowest divided, monotone between; the size of the values
    yarn = rope.rotary_table(2, 64, 1e4, dict(type="yarn", factor=8.0, original=4096), dtype=torch.float64)
    angle = torch.atan2(yarn[1, 32:], yarn[1, :32])
    base = 1e4 ** (-torch.arange(32).double() / 32)
    share = base / angle
    turns = 4096 * base / (2 * math.pi)
    assert torch.allclose(share[turns > 64], torch.ones((), dtype=torch.float64), atol=1e-9)
    assert torch.allclose(share[turns < 0.5], torch.full((), 8.0, dtype=torch.float64), atol=1e-9)
    assert bool((share[1:] >= share[:-1] - 1e-9).all())
    assert math.isclose(float(yarn[0, 0]), 0.1 * math.log(8.0) + 1, rel_tol=1e-12)
    own = dict(type="yarn", factor=8.0, original=4096, beta_fast=16, beta_slow=2, attention_factor=1.0)
    assert float(rope.rotary_table(2, 64, 1e4, own)[0, 0]) == 1.0


@pytest.mark.parametrize("args,scaling", [
    ((0, 64, 1e4), None), ((4, 63, 1e4), None), ((4, 64, 0.0), None), ((4, 64, 1e4), dict(type="other", factor=2.0)),
    ((4, 64, 1e4), dict(type="linear", factor=0.5)), ((4, 64, 1e4), dict(type="yarn", factor=2.0)),
    ((4, 64, 1e4), dict(type="linear", factor=2.0, original=4)), ((4, 64, 1e4), dict(factor=2.0)),
    ((4, 2, 1e4), dict(type="ntk", factor=2.0))])
def test_rotary_tables_refused(args, scaling):
    with pytest.raises(ValueError):
        rope.rotary_table(*args, scaling)


# ------------------------------------------------------------------- C ABI --

def packed(name, values):
    """The arguments' struct: every field takes 8 bytes, in the header's order."""
    return _lib._STRUCTS[name].pack(*[0 if x is None else x for x in values])


def rotate(h, q=_P, v=_P, cos=_P, table_len=16, rotary=64, pos=_P, k_pages=_P, v_pages=_P, table=_P, batch=2, width=4,
           pages=8, page=16, rows=3, hq=4, hkv=2, dim=64, qs=64, q_out=_P, k_out=None):
    return h.lm_paged_rotate_write(packed("lm_paged_rotate_write", [
        q, qs, 64, _P, 64, 64, v, 64, 64, cos, table_len, rotary, 1, 1, pos, None, 0, None, None, q_out, 64, 64, k_out, 64,
        64, k_pages, v_pages, table, batch, width, pages, page, rows, hq, hkv, dim]), None)


def read(h, k=_P, page=16, dim=64, rows=3, table=_P, out=_P):
    return h.lm_paged_read(packed("lm_paged_read", [k, _P, table, 2, 4, 8, page, _P, 0, None, rows, 2, dim, out, _P]), None)


def decode(h, q=_P, page=16, width=4, pages=8, batch=2, hq=4, hkv=2, dim=64, max_len=64, splits=1, shares=0, w=None, w_out=None,
           ws=_P, size=1 << 30, table=_P, qs=64):
    return h.lm_flash_decode_paged(packed("lm_flash_decode_paged", [
        q, qs, 64, _P, _P, table, width, pages, page, _P, batch, hq, hkv, dim, 1.0, max_len, splits, shares, w, w_out, _P, ws,
        size]), None)


def fused(h, part=_P, slices=3, cos=_P, rotary=64, page=16, batch=2, frag=0, pos=_P, ws=_P, size=1 << 30, splits=1):
    return h.lm_flash_decode_paged_qkv(packed("lm_flash_decode_paged_qkv", [
        part, slices, cos, 16, rotary, 1, 1, pos, None, _P, _P, _P, 4, 8, page, _P, None, batch, 4, 2, 64, 1.0, 64, splits,
        None, None, frag, _P, ws, size]), None)


def evict(h, page=16, keep=5, recent=2, layers=2, batch=2, width=4, w=_P, dim=64, target=_P):
    return h.lm_kv_evict(packed("lm_kv_evict", [
        _P, _P, _P, target, width, 2, 8, page, _P, w, layers, batch, 2, dim, keep, recent, _P, _P, _P]), None)


@pytest.mark.parametrize("name", ["lm_paged_rotate_write", "lm_paged_read", "lm_kv_evict", "lm_flash_decode_paged",
                                  "lm_flash_decode_paged_qkv"])
def test_structs_are_the_headers(name):
    """Fields and their kinds, in order; no struct at all is refused."""
    text = (Path(__file__).resolve().parents[1] / "include" / "litemoe_amd.h").read_text()
    tag = name.replace("_write", "") + "_args"
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (tag, tag), text, re.S).group(1)
    kinds = ""
    for line in body.split(";")[:-1]:
        count = line.count(",") + 1
        assert "*" in line or re.match(r"\s*(int64_t|double) ", line), line
        kinds += ("d" if line.split()[0] == "double" else "q") * count
    fields = _lib._STRUCTS[name].format
    assert kinds == "".join(kind * int(n or 1) for n, kind in re.findall(r"(\d*)([qd])", fields))
    assert _lib._STRUCTS[name].size == 8 * len(kinds)
    assert getattr(_lib.load(), name)(None, None) == 1


@pytest.mark.parametrize("call,expected", [
    (lambda h: rotate(h, rows=0), 0), (lambda h: rotate(h, rows=-1), 1), (lambda h: rotate(h, page=24), 2),
    (lambda h: rotate(h, page=8), 2), (lambda h: rotate(h, dim=96), 2), (lambda h: rotate(h, dim=72), 2),
    (lambda h: rotate(h, v_pages=None), 1), (lambda h: rotate(h, table=None), 1), (lambda h: rotate(h, v=None), 1),
    (lambda h: rotate(h, rotary=24), 1), (lambda h: rotate(h, rotary=80), 1), (lambda h: rotate(h, rotary=0), 1),
    (lambda h: rotate(h, cos=None), 1), (lambda h: rotate(h, pos=None), 1), (lambda h: rotate(h, q=_P + 2), 1),
    (lambda h: rotate(h, qs=60), 1), (lambda h: rotate(h, q_out=None), 1), (lambda h: rotate(h, table_len=0), 1),
    (lambda h: rotate(h, width=0), 1), (lambda h: rotate(h, pages=0), 1), (lambda h: rotate(h, pages=1 << 31), 1),
    (lambda h: rotate(h, width=1 << 27), 1), (lambda h: rotate(h, batch=0), 1), (lambda h: rotate(h, rows=1 << 40), 1),
    (lambda h: rotate(h, k_pages=None, v_pages=None), 1),  # neither k_out nor a cache
    (lambda h: read(h, rows=0), 0), (lambda h: read(h, page=48), 2), (lambda h: read(h, dim=32), 2),
    (lambda h: read(h, table=None), 1), (lambda h: read(h, out=_P + 8), 1), (lambda h: read(h, rows=1 << 40), 1),
    (lambda h: decode(h, batch=0), 0), (lambda h: decode(h, hq=5), 1), (lambda h: decode(h, hq=34), 2),
    (lambda h: decode(h, dim=96), 2), (lambda h: decode(h, page=17), 2), (lambda h: decode(h, q=None), 1),
    (lambda h: decode(h, q=_P + 4), 1), (lambda h: decode(h, qs=65), 1), (lambda h: decode(h, table=None), 1),
    (lambda h: decode(h, max_len=0), 1), (lambda h: decode(h, splits=0), 1), (lambda h: decode(h, splits=1025), 1),
    (lambda h: decode(h, shares=-1), 1), (lambda h: decode(h, shares=65536), 1), (lambda h: decode(h, splits=2, shares=2), 1),
    (lambda h: decode(h, w=_P), 1), (lambda h: decode(h, w_out=_P), 1), (lambda h: decode(h, w=_P + 4, w_out=_P), 1),
    (lambda h: decode(h, shares=2, size=100), 4), (lambda h: decode(h, shares=2, w=_P, w_out=_P, ws=None), 4),
    (lambda h: decode(h, shares=2, ws=_P + 4), 1), (lambda h: decode(h, splits=2, size=100), 4),
    (lambda h: decode(h, w=_P, w_out=_P, max_len=15361, width=300, size=100), 4), (lambda h: decode(h, batch=65536), 1),
    (lambda h: fused(h, batch=0), 0), (lambda h: fused(h, slices=9), 2), (lambda h: fused(h, slices=0), 1),
    (lambda h: fused(h, rotary=72), 1), (lambda h: fused(h, cos=None), 1), (lambda h: fused(h, part=_P + 4), 1),
    (lambda h: fused(h, batch=129, frag=1), 2), (lambda h: fused(h, pos=None), 1), (lambda h: fused(h, page=20), 2),
    (lambda h: fused(h, splits=2, size=8), 4),
    (lambda h: evict(h, batch=0), 0), (lambda h: evict(h, keep=0), 1), (lambda h: evict(h, recent=6), 1),
    (lambda h: evict(h, recent=-1), 1), (lambda h: evict(h, keep=65), 1), (lambda h: evict(h, page=15), 2),
    (lambda h: evict(h, w=None), 1), (lambda h: evict(h, layers=0), 1), (lambda h: evict(h, layers=300, batch=300), 1),
    (lambda h: evict(h, dim=80), 2), (lambda h: evict(h, target=None), 1), (lambda h: evict(h, w=_P + 8), 1),
    (lambda h: evict(h, width=769), 1),  # in place, rows of more than 12288 positions
])
def test_invalid_arguments_rejected_on_host(call, expected):
    assert call(_lib.load()) == expected


def test_workspace_sizes():
    def size(splits, shares, weighed, max_len=100):
        return _lib.size_query("lm_flash_decode_paged_workspace_size", 3, 8, 2, 128, max_len, splits, shares, weighed)
    assert size(1, 0, 0) == size(1, 0, 1) == 0
    assert size(4, 0, 0) == 3 * 4 * 8 * 128 * 4 + 2 * 512
    assert size(1, 5, 0) == 256 + 5 * 8 * 2 * 128 * 4 + 2 * 512
    scores = 2 * 256 + 3 * 8 * 128 * 4
    assert size(4, 0, 1) == size(4, 0, 0) + scores and size(1, 5, 1) == size(1, 5, 0) + scores
    # four query heads' scores of 7712 positions are more than a workgroup keeps
    assert size(1, 0, 1, 7680) == 0 and size(1, 0, 1, 7681) == 2 * 256 + 3 * 8 * 7712 * 4


# ------------------------------------------------------------------ oracle --

def test_oracle_against_dense_torch():
    """The oracle's rows, attention, rotation and choice against torch on a dense cache."""
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(6, 2, 16, 64, generator=g).to(torch.bfloat16) for _ in range(2))
    table = torch.tensor([[3, 0, 5], [1, -1, 2]], dtype=torch.int32)
    q = torch.randn(2, 4, 64, generator=g).to(torch.bfloat16)
    out, p = paged.attention(q, k, v, table, [40, 48], 0.125)
    dense_k, dense_v = (torch.cat([x[i] for i in (3, 0, 5)], 1)[:, :40].double() for x in (k, v))
    s = q[0].double().view(2, 2, 64) @ dense_k.transpose(1, 2) * 0.125
    assert torch.allclose(out[0].view(2, 2, 64), torch.softmax(s, -1) @ dense_v, atol=1e-12)
    assert p[1].shape == (2, 2, 48) and bool((p[1][:, :, 16:32] == 0).all())
    assert torch.allclose(p[1].sum(-1), torch.ones(2, 2, dtype=torch.float64))
    pos = torch.tensor([0, 5, 77])
    cos, sin = paged.angles(pos, 64, 1e4)
    x = torch.randn(3, 2, 64, generator=g).double()
    half = torch.cat((-x[..., 32:], x[..., :32]), -1)
    c2, s2 = (torch.cat((a, a), -1)[:, None] for a in (cos, sin))
    assert torch.allclose(paged.rotate(x, cos, sin, True), x * c2 + half * s2, atol=1e-12)
    inter = paged.rotate(x, cos, sin, False)
    z = torch.view_as_complex(x.view(3, 2, 32, 2).contiguous()) * torch.polar(torch.ones_like(cos), torch.atan2(
        sin, cos))[:, None]
    assert torch.allclose(inter, torch.view_as_real(z).flatten(-2), atol=1e-12)
    w = torch.tensor([1.0, 3.0, 2.0, 3.0, 0.5, 9.0])
    assert paged.keep(w, 6, 3, 1) == [1, 3, 5] and paged.keep(w, 6, 2, 2) == [4, 5] and paged.keep(w, 2, 3, 0) == [0, 1]
    assert paged.keep(torch.tensor([1.0, math.nan, 1.0]), 3, 2, 0) == [0, 1]
