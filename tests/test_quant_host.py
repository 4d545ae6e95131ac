"""The quantised KV cache without a GPU: its number format, its buffers, and
the calls that are refused before anything is launched."""
import copy
import ctypes as C
import math
import pickle

import pytest
import torch

from litemoe_amd import _lib, kv_quant
from litemoe_amd.cache import KVCache, QuantKVCache
from litemoe_amd.config import preset
from litemoe_amd.engine import Engine
from litemoe_amd.flash_decode import QuantFlashDecode, quant_splits
from litemoe_amd.linear import linear_rope_kv
from oracle import quant

_P = 1 << 20


def test_lists_of_values_are_the_types():
    """The oracle's lists against the bit fields: torch's own 8-bit type, and
    the 4-bit values by sign, exponent and mantissa."""
    e4m3 = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    assert torch.equal(quant.grid(8), e4m3)
    for c, value in enumerate(quant.E2M1):
        e, m = c >> 1, c & 1
        assert value == ((1 + m / 2) * 2.0 ** (e - 1) if e else m / 2)


@pytest.mark.parametrize("bits", [4, 8])
def test_oracle_error_is_the_types(bits):
    """Every element within half a step of the type's grid, of the block's
    largest value where that is held: a quarter of the scale's unit at least
    (half the smallest step) and 2^-2 (4 bits) or 2^-4 (8) of the value."""
    x = (3 * torch.randn(40, 64, generator=torch.Generator().manual_seed(bits))).to(torch.bfloat16)
    codes, scales = quant.quantise(x, bits)
    back = quant.values(codes, scales, bits)
    unit = 2.0 ** (scales.double() - 127).repeat_interleave(32, -1)
    relative, least = (0.25, 0.25) if bits == 4 else (2.0 ** -4, 2.0 ** -10)
    assert bool(((back - x.double()).abs() <= torch.maximum(relative * x.double().abs(), least * unit)).all())
    # the rule's two edges: T 2^e keeps e, the next bf16 above takes e + 1
    for top, byte in ((quant.TOP[bits], 127), (quant.TOP[bits] * (1 + 2.0 ** -6), 128)):
        block = torch.zeros(64, dtype=torch.float64)
        block[5] = top
        assert quant.quantise(block, bits)[1][0] == byte
    # codes pack and unpack; a quantised vector quantises to itself
    assert torch.equal(quant.unpack(quant.pack(codes, bits), bits), codes)
    again, _ = quant.quantise(back, bits)
    assert torch.equal(quant.values(again, quant.quantise(back, bits)[1], bits), back)


def test_cache_buffers_and_bytes():
    cfg = preset("granite-3b", num_hidden_layers=2)
    plain = KVCache(cfg, 3, 40, "cpu", torch.bfloat16)
    for bits, per_position in ((4, 68), (8, 132)):
        cache = QuantKVCache(cfg, 3, 40, "cpu", torch.bfloat16, bits=bits)
        assert cache.bits == bits and cache.capacity == 40
        total = sum(t.numel() for t in (cache.k, cache.v, cache.scales))
        assert total == 2 * 3 * 8 * 40 * per_position
        assert total * 256 == per_position * 2 * (plain.k.numel() + plain.v.numel())
        assert all(not bool(t.any()) for t in (cache.k, cache.v, cache.scales))
        layer = cache.layer(1)
        assert layer.k.data_ptr() == cache.k[1].data_ptr() and layer.scales.shape == (3, 8, 40, 4)
        cache.k.fill_(7), cache.v.fill_(7), cache.scales.fill_(7)
        cache.clear(1, 4, 9)
        for t in (cache.k, cache.v, cache.scales):
            assert not bool(t[:, 1, :, 4:9].any()) and bool((t[:, 1, :, 9:] == 7).all()) and bool((t[:, 0] == 7).all())
        cache.reset()
        assert not bool(cache.scales.any())
        over = QuantKVCache.over(cache.k, cache.v, cache.scales)
        assert over.k is cache.k and over.bits == bits and over.capacity == 40


@pytest.mark.parametrize("slot,rows", [(1, 1), (slice(0, 2), 2)])
def test_prefill_by_rows_of_a_quantised_cache(slot, rows, monkeypatch):
    """A quantised cache's rows share nothing: a prefill by rows stores every position of them."""
    stored = []
    monkeypatch.setattr(kv_quant, "write", lambda cache, layer, k, v, at, active, slots: stored.extend(
        zip(slots.tolist(), at.tolist())))
    cfg = preset("granite-1b", num_hidden_layers=1)
    cache = QuantKVCache(cfg, 2, 16, "cpu", torch.bfloat16)
    x = torch.zeros(rows, cfg.num_key_value_heads, 3, 64, dtype=torch.bfloat16)
    cache.prefill(0, slot, x, x, torch.ones(rows, 3, dtype=torch.bool))
    assert stored == [(row, j) for row in (range(2) if rows == 2 else [1]) for j in range(3)]


def test_python_refusals():
    cfg = preset("granite-1b", num_hidden_layers=1)
    with pytest.raises(ValueError, match="4 or 8 bits"):
        QuantKVCache(cfg, 1, 16, "cpu", torch.bfloat16, bits=2)
    with pytest.raises(ValueError, match="BF16"):
        QuantKVCache(cfg, 1, 16, "cpu", torch.float32)
    with pytest.raises(ValueError, match="head_dim 64"):
        QuantKVCache(preset("granite-1b", num_hidden_layers=1, num_attention_heads=8), 1, 16, "cpu", torch.bfloat16)
    cache = QuantKVCache.empty(1, 2, 2, 16, "cpu", bits=4)
    with pytest.raises(ValueError, match="Quantised KV buffers are"):
        QuantKVCache.over(cache.k, cache.v[..., :16], cache.scales)
    with pytest.raises(ValueError, match="contiguous uint8"):
        QuantKVCache.over(cache.k, cache.v, cache.scales.to(torch.int32))
    x = torch.zeros(2, 2, 1, 64, dtype=torch.bfloat16)
    pos, act = torch.zeros(2, dtype=torch.long), torch.ones(2, dtype=torch.bool)
    with pytest.raises(ValueError, match="no CPU fallback"):
        cache.write(0, x, x, pos, act)
    with pytest.raises(ValueError, match="no CPU fallback"):
        kv_quant.read(cache, 0, pos, pos)
    for bad in (dict(bits=5), dict(maximum=17), dict(maximum=0), dict(groups=17), dict(groups=0)):
        args = dict(batch=1, kv_heads=2, groups=3, capacity=16, device="cpu")
        with pytest.raises(ValueError):
            QuantFlashDecode(**{**args, **bad})
    flash = QuantFlashDecode(2, 2, 1, 16, "cpu", bits=4)
    with pytest.raises(ValueError, match="no CPU fallback"):
        flash(x, *cache.layer(0), pos, act, 0.125)
    with pytest.raises(ValueError, match="16 bits per element"):
        Engine(None, [], kv_bits=5)
    with pytest.raises(ValueError, match="no CPU fallback"):
        linear_rope_kv(x[:, 0, 0], x[:, 0, 0], 1, 1, pos, None, x[:, 0, 0], None, 0)


def _write(h, **over):
    a = dict(k=_P, ks=(128, 64, 1), v=_P, kc=_P, vc=_P, sc=_P, pos=_P, rows=4, heads=2, d=64, cap=16, batch=4, bits=4)
    a.update(over)
    return h.lm_kv_quant_write(a["k"], *a["ks"], a["v"], *a["ks"], a["kc"], a["vc"], a["sc"], a["pos"], None, None,
                               a["rows"], a["heads"], a["d"], a["cap"], a["batch"], a["bits"], None)


def _read(h, **over):
    a = dict(kc=_P, vc=_P, sc=_P, pos=_P, rows=4, heads=2, d=64, cap=16, batch=4, bits=4, k=_P, v=_P)
    a.update(over)
    return h.lm_kv_quant_read(a["kc"], a["vc"], a["sc"], a["pos"], None, a["rows"], a["heads"], a["d"], a["cap"],
                              a["batch"], a["bits"], a["k"], a["v"], None)


def _decode(h, **over):
    a = dict(q=_P, qs=(128, 64), kc=_P, vc=_P, sc=_P, used=_P, batch=2, hq=4, hkv=2, cap=128, d=64, bits=4, max=128,
             splits=2, out=_P, ws=_P, size=1 << 30)
    a.update(over)
    return h.lm_flash_decode_quant(a["q"], *a["qs"], a["kc"], a["vc"], a["sc"], a["used"], a["batch"], a["hq"],
                                   a["hkv"], a["cap"], a["d"], a["bits"], C.c_float(0.125), a["max"], a["splits"],
                                   a["out"], a["ws"], a["size"], None)


def _fused(h, **over):
    a = dict(part=_P, qkv=3, cs=_P, table=128, pos=_P, kc=_P, vc=_P, sc=_P, used=_P, batch=2, hq=4, hkv=2, cap=128,
             d=64, bits=8, max=128, splits=2, frag=0, out=_P, ws=_P, size=1 << 30)
    a.update(over)
    return h.lm_flash_decode_quant_qkv(a["part"], a["qkv"], a["cs"], a["table"], a["pos"], None, a["kc"], a["vc"],
                                       a["sc"], a["used"], None, a["batch"], a["hq"], a["hkv"], a["cap"], a["d"],
                                       a["bits"], C.c_float(0.125), a["max"], a["splits"], a["frag"], a["out"],
                                       a["ws"], a["size"], None)


_COMMON = [(dict(bits=5), 2), (dict(d=128), 2), (dict(cap=0), 1), (dict(kc=_P + 8), 1), (dict(vc=None), 1),
           (dict(sc=_P + 2), 1)]


@pytest.mark.parametrize("call,over,expected", [
    *[(f, *c) for f in (_write, _read, _decode, _fused) for c in _COMMON],
    *[(f, *c) for f in (_write, _read) for c in [
        (dict(rows=-1), 1), (dict(rows=(1 << 28) + 1), 1), (dict(heads=0), 1), (dict(heads=65536), 1),
        (dict(batch=0), 1), (dict(pos=None), 1), (dict(rows=0, pos=None, kc=None), 0), (dict(k=None), 1)]],
    (_write, dict(k=_P + 1), 1), (_read, dict(v=_P + 8), 1),
    *[(f, *c) for f in (_decode, _fused) for c in [
        (dict(batch=-1), 1), (dict(batch=65536), 1), (dict(hq=5), 1), (dict(hq=34, hkv=2), 2), (dict(max=0), 1),
        (dict(max=1 << 30), 1), (dict(splits=0), 1), (dict(splits=1025), 1), (dict(used=None), 1),
        (dict(out=None), 1), (dict(ws=None), 4), (dict(size=16), 4), (dict(ws=_P + 4), 1),
        (dict(batch=0, used=None), 0)]],
    (_decode, dict(q=None), 1), (_decode, dict(q=_P + 8), 1), (_decode, dict(qs=(128, 60)), 1),
    (_fused, dict(qkv=0), 1), (_fused, dict(qkv=9), 2), (_fused, dict(table=0), 1), (_fused, dict(cs=None), 1),
    (_fused, dict(part=_P + 4), 1), (_fused, dict(frag=1, batch=129), 2), (_fused, dict(pos=None), 1),
])
def test_status_codes_before_launch(call, over, expected):
    """Refused on the host (LM_EINVAL 1, LM_EUNSUPPORTED 2, LM_EWORKSPACE 4), or
    nothing to do (0): no case here launches a kernel."""
    assert call(_lib.load(), **over) == expected


def test_oracle_attention_of_an_empty_row_and_of_one_position():
    g = torch.Generator().manual_seed(5)
    q, k, v = torch.randn(2, 4, 64, generator=g), *torch.randn(2, 2, 2, 8, 64, generator=g)
    out = quant.decode_attention(q, k, v, torch.tensor([0, 1]), 1 / math.sqrt(64))
    assert not bool(out[0].any())
    assert torch.allclose(out[1], v[1, :, 0].repeat_interleave(2, 0).double())


@pytest.mark.parametrize("batch,kv_heads,maximum,splits", [
    (1, 8, 1, 1), (1, 8, 1535, 1), (1, 8, 1536, 3), (1, 8, 4000, 8), (3, 8, 4001, 8), (5, 8, 4000, 6), (8, 8, 8191, 4),
    (8, 8, 8192, 8), (20, 8, 16000, 8), (40, 8, 8192, 8), (32, 8, 32768, 1), (41, 8, 32768, 1), (16, 8, 4095, 2), (17, 8, 4095, 1), (32, 8, 4095, 1), (64, 8, 1279, 1), (128, 8, 4096, 1), (1, 1, 32768, 16),
    (1, 1, 1 << 20, 256)])
def test_quant_splits(batch, kv_heads, maximum, splits):
    assert quant_splits(batch, kv_heads, maximum) == splits


def test_quant_splits_fill_the_cus_and_keep_512_positions():
    for batch in (1, 2, 5, 16, 31, 33, 200):
        for maximum in (1, 511, 1536, 4096, 32768, 1 << 20):
            n = quant_splits(batch, 8, maximum)
            assert n >= 1 and (n == 1 or -(-maximum // n) > 512 - 64)
            assert n * batch * 8 <= 256 or n == 1 or (n == 8 and maximum >= 8192)


@pytest.mark.parametrize("maximum", [8192, 16000, 32768, 1 << 20])
def test_quant_splits_of_long_contexts_go_by_ranges(maximum):
    """One split where the pairs leave less than an eighth of the CUs free or are too many
    to gain, eight or more elsewhere: no number of pairs stands apart from its neighbours."""
    for pairs in range(1, 600):
        n = quant_splits(pairs, 1, maximum)
        assert (n == 1) if 224 < pairs <= 256 or pairs > 320 else n >= 8
    for batch in (29, 31, 32, 33):
        assert quant_splits(batch, 8, maximum) == quant_splits(8 * batch, 1, maximum)


def test_layers_are_views_of_the_buffers_the_cache_holds():
    """Buffers replaced by others, a copy and a pickled cache: ``layer`` gives views of what
    ``k``, ``v`` and ``scales`` are, as a KVCache's own indexing does."""
    cache = QuantKVCache.empty(2, 3, 2, 16, "cpu", bits=4)
    cache.layer(0)
    fresh = [torch.full_like(t, 3) for t in (cache.k, cache.v, cache.scales)]
    cache.k, cache.v, cache.scales = fresh
    for other in (cache, copy.copy(cache), copy.deepcopy(cache), pickle.loads(pickle.dumps(cache))):
        for layer in range(2):
            held = other.layer(layer)
            assert [t.data_ptr() for t in held] == [t[layer].data_ptr() for t in (other.k, other.v, other.scales)]
            assert all(bool((t == 3).all()) for t in held)
        assert other.bits == 4 and other.capacity == 16
    assert copy.deepcopy(cache).k.data_ptr() != cache.k.data_ptr()
    for bad in (fresh[0][:1], fresh[0].int(), fresh[0].transpose(1, 2)):
        with pytest.raises(ValueError, match="same shape, type and device"):
            cache.k = bad
    assert cache.k is fresh[0]
