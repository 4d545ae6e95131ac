"""The quantised KV cache on the GPU: store, read-back and decode attention
against the oracle in 64 bits (oracle/quant.py).

Codes, scale bytes and read-back values are exact. The attention's tolerance is
derived per element (:func:`bound`).
"""
import pytest
import torch

from litemoe_amd import kv_quant, synth
from litemoe_amd.batch import BatchPrefillEngine
from litemoe_amd.cache import KVCache, QuantKVCache
from litemoe_amd.config import preset
from litemoe_amd.engine import Engine, Request
from litemoe_amd.ep import ExpertParallel
from litemoe_amd.execution import capture_decode
from litemoe_amd.experts import HipFusedExperts
from litemoe_amd.flash_decode import FlashDecode, QuantFlashDecode
from litemoe_amd.linear import linear_dense, linear_rope_kv, linear_splitk, linear_splitk_frag
from litemoe_amd.model import Granite
from litemoe_amd.optimized import OptimizedEngine
from litemoe_amd.packed import build_packed
from litemoe_amd.rope import rotary_embedding
from oracle import ops, quant

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16


def gen(seed):
    return torch.Generator().manual_seed(seed)


def vectors(shape, seed):
    """bf16 vectors whose channels have unequal sizes."""
    g = gen(seed)
    return (torch.randn(shape, generator=g) * torch.exp(0.5 * torch.randn(shape[-1], generator=g))).to(BF16)


def random_cache(bits, batch, heads, capacity, seed, layers=1):
    """A cache of quantised vectors, and the values it stands for (64 bits, CPU)."""
    cache = QuantKVCache.empty(layers, batch, heads, capacity, DEV, bits=bits)
    # vectors drawn from a pool, so that the oracle quantises few
    pool = 193
    sides = []
    for side, seed_at in ((cache.k, 0), (cache.v, 1)):
        codes, scales = quant.quantise(vectors((pool, 64), seed + seed_at), bits)
        index = torch.randint(0, pool, (layers, batch, heads, capacity), generator=gen(seed + 7 + seed_at))
        side.copy_(quant.pack(codes, bits)[index])
        cache.scales[..., 2 * seed_at:2 * seed_at + 2].copy_(scales.to(torch.uint8)[index])
        sides.append(quant.values(codes, scales, bits)[index])
    return cache, *sides


def bound(q, k, v, used, scale, out):
    """How far a row's outputs may be from the exact ones, per element, with
    A = sum p|v| / sum p:
    * probabilities are rounded to bf16, p(1 + d) with |d| <= 2^-8, and summed as
      rounded (V's scale is a power of two and adds no rounding):
      sum p(1 + d)v / sum p(1 + d) - out = sum pd(v - out) / sum p(1 + d), at most
      2^-8 (A + |out|) / (1 - 2^-8); the result's own rounding adds 2^-8 of it. Together
      less than 2^-8 (1 + 2^-6) (A + 2|out|);
    * a score is a sum of 64 products in fp32 with 64 + 8 roundings of at most
      2^-24 of sum|q k|; that moves p by the same share, in numerator and
      denominator, and the sums over n positions (in any order, with the
      exponential's and the merges' few roundings) add (n + 64) 2^-24 of
      A + |out| each."""
    b, hq, _ = q.shape
    hkv = k.shape[1]
    tol = torch.zeros(out.shape, dtype=torch.float64)
    for i in range(b):
        n = max(0, min(int(used[i]), k.shape[2]))
        if not n:
            continue
        qi = q[i].double().view(hkv, hq // hkv, 64)
        ki, vi = k[i, :, :n].double(), v[i, :, :n].double()
        p = torch.softmax(qi @ ki.transpose(1, 2) * scale, -1)
        a = (p @ vi.abs()).reshape(hq, 64)
        size = (qi.abs() @ ki.abs().transpose(1, 2)).amax(-1).reshape(hq, 1) * scale
        o = out[i].abs()
        tol[i] = 2.0 ** -8 * (1 + 2.0 ** -6) * (a + 2 * o) + 2.0 ** -24 * (2 * 72 * size + n + 64) * (a + o)
    return tol + 1e-30


def check(got, q, k, v, used, scale):
    exp = quant.decode_attention(q, k, v, used, scale)
    over = ((got.double().cpu() - exp).abs() - bound(q, k, v, used, scale, exp)).amax()
    assert float(over) <= 0, float(over)


# ------------------------------------------------------------ store, read --

@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("rows,heads,capacity", [(1, 1, 1), (5, 2, 33), (33, 8, 64), (64, 3, 40)])
@torch.inference_mode()
def test_store_and_read_back(bits, rows, heads, capacity):
    x = [vectors((rows, heads, 64), 3 * rows + i) for i in range(2)]
    batch = 3
    cache = QuantKVCache.empty(2, batch, heads, capacity, DEV, bits=bits)
    for t in (cache.k, cache.v, cache.scales):
        t.copy_(torch.randint(0, 256, t.shape, generator=gen(rows), dtype=torch.uint8))
    # distinct targets, some of them out of range or inactive
    at = torch.randperm(batch * capacity, generator=gen(rows + 1))[:rows]
    at = torch.cat((at, -torch.ones(rows - at.numel(), dtype=torch.long)))
    slots, positions = at // capacity, at % capacity
    slots[at < 0], positions[at < 0] = batch, 0
    if rows > 4:
        positions[1], positions[2] = capacity, -1
    active = torch.ones(rows, dtype=torch.bool)
    active[3::7] = False
    before = [t.cpu() for t in (cache.k, cache.v, cache.scales)]
    cache.write(1, x[0].to(DEV)[:, :, None], x[1].to(DEV)[:, :, None], positions.to(DEV), active.to(DEV), slots.to(DEV))
    inside = (positions >= 0) & (positions < capacity) & (slots >= 0) & (slots < batch)
    expected = [t.clone() for t in before]
    want = []
    for side, (v, t) in enumerate(zip(x, expected)):
        codes, scales = quant.quantise(v, bits)
        for r in range(rows):
            if active[r] and inside[r]:
                t[1, slots[r], :, positions[r]] = quant.pack(codes[r], bits)
                expected[2][1, slots[r], :, positions[r], 2 * side:2 * side + 2] = scales[r].to(torch.uint8)
        want.append(quant.values(codes, scales, bits))
    for got, exp in zip((cache.k, cache.v, cache.scales), expected):
        assert torch.equal(got.cpu(), exp)
    back = kv_quant.read(cache, 1, positions.to(DEV), slots.to(DEV))
    for got, exp in zip(back, want):
        got = got[:, :, 0].cpu()
        stored = active & inside
        assert torch.equal(got[stored].double(), exp[stored])
        assert not bool(got[~inside].any())


@pytest.mark.parametrize("bits", [4, 8])
@torch.inference_mode()
def test_store_of_every_kind_of_block(bits):
    """Blocks of zeros, of the smallest and largest numbers, at the rounding's
    ties and the scale rule's edges, with infinities and NaN; one block of a
    vector does not touch the other."""
    g = gen(bits)
    top = quant.TOP[bits]
    blocks = [torch.zeros(32), torch.full((32,), -0.0), torch.randn(32, generator=g) * 2.0 ** -130,
              torch.full((32,), 2.0 ** -133), torch.randn(32, generator=g).clamp(-1.9, 1.9) * 2.0 ** 127,
              torch.full((32,), 3.3895e38), torch.linspace(-top, top, 32), torch.linspace(0, 2, 32) * 2.0 ** 40,
              torch.arange(32) * 0.25, torch.arange(32) * -0.125,
              torch.cat((torch.tensor([top]), torch.rand(31, generator=g))),
              torch.cat((torch.tensor([top * 1.01]), torch.rand(31, generator=g))), torch.full((32,), top * 2.0 ** 118),
              torch.cat((torch.tensor([1.0]), torch.full((31,), 2.0 ** -12)))]
    grid = quant.grid(bits)
    ties = (grid[1:] + grid[:-1]) / 2
    for part in ties.split(31):
        blocks.append(torch.cat((torch.tensor([top]), part.float(), torch.zeros(31 - part.numel()))))
    special = []
    for bad in (float("inf"), -float("inf"), float("nan")):
        block = torch.randn(32, generator=g)
        block[17] = bad
        special.append(block)
    pairs = [torch.cat((a, b)) for a, b in zip(blocks, blocks[1:] + blocks[:1])]
    pairs += [torch.cat((s, blocks[9])) for s in special] + [torch.cat((blocks[10], s)) for s in special]
    x = torch.stack(pairs).to(BF16)
    rows = x.shape[0]
    cache = QuantKVCache.empty(1, 1, 1, rows, DEV, bits=bits)
    every = torch.arange(rows, device=DEV)
    zero = torch.zeros_like(every)
    cache.write(0, x.to(DEV)[:, None, None], x.flip(1).contiguous().to(DEV)[:, None, None], every, None, zero)
    for got, codes_got, part, v in ((kv_quant.read(cache, 0, every, zero)[0], cache.k, slice(0, 2), x),
                                    (kv_quant.read(cache, 0, every, zero)[1], cache.v, slice(2, 4), x.flip(1))):
        codes, scales = quant.quantise(v, bits)
        assert torch.equal(codes_got[0, 0, 0].cpu(), quant.pack(codes, bits))
        assert torch.equal(cache.scales[0, 0, 0, :, part].cpu().long(), scales)
        want = quant.values(codes, scales, bits)
        got = got[:, 0, 0].cpu()
        nan = want.isnan()
        assert torch.equal(got.isnan(), nan)
        assert torch.equal(got[~nan].double(), want[~nan])


@pytest.mark.parametrize("bits", [4, 8])
@torch.inference_mode()
def test_store_takes_any_strides(bits):
    """Head and row strides, an offset that is not 16-byte aligned, channels
    that are not contiguous, one row broadcast to all heads."""
    rows, heads = 21, 4
    base = vectors((rows, 2, heads, 70), 5).to(DEV)
    odd = base.flatten()[1:1 + rows * 560 - 560].unfold(0, 64, 70)[:rows * heads].view(rows, heads, 1, 64)
    views = [base[:, 0, :, 3:67].unsqueeze(2), base[:, 1, :, :64].unsqueeze(2), odd,
             base[:, 0, :, :64].transpose(1, 2).contiguous().transpose(1, 2).unsqueeze(2),
             base[:, 0, :1, :64].expand(rows, heads, 64).unsqueeze(2)]
    every = torch.arange(rows, device=DEV)
    for k, v in zip(views, views[1:] + views[:1]):
        cache = [QuantKVCache.empty(1, rows, heads, 2, DEV, bits=bits) for _ in range(2)]
        cache[0].write(0, k, v, torch.ones_like(every), None)
        cache[1].write(0, k.contiguous(), v.contiguous(), torch.ones_like(every)[:, None], None)
        assert bool(cache[0].scales.any())
        for a, b in zip(cache[0].layer(0), cache[1].layer(0)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("bits", [4, 8])
@torch.inference_mode()
def test_cache_prefill_decode_and_read(bits):
    """The KVCache interface: a padded prefill, a packed one and a decode step
    against the bf16 cache's, quantised."""
    cfg = preset("granite-1b", num_hidden_layers=1)
    b, s, cap = 3, 11, 24
    cache, plain = QuantKVCache(cfg, b, cap, DEV, BF16, bits=bits), KVCache(cfg, b, cap, DEV, BF16)
    k, v = (vectors((b, 8, s, 64), i).to(DEV) for i in range(2))
    lengths = torch.tensor([11, 4, 0], device=DEV)
    valid = torch.arange(s, device=DEV)[None] < lengths[:, None]
    got, exp = cache.prefill(0, slice(0, b), k, v, valid), plain.prefill(0, slice(0, b), k, v, valid)
    assert all(torch.equal(x, y) for x, y in zip(got, exp))
    packed, _ = build_packed([5, 2], DEV, slots=[1, 2])
    kp, vp = (vectors((1, 8, 7, 64), 9 + i).to(DEV) for i in range(2))
    assert cache.prefill(0, packed, kp, vp, None)[2] is None and plain.prefill(0, packed, kp, vp, None)[2] is None
    active = torch.tensor([True, True, False], device=DEV)
    kn, vn = (vectors((b, 8, 1, 64), 19 + i).to(DEV) for i in range(2))
    gk, gv, gm = cache.decode(0, kn, vn, lengths, active)
    ek, ev, em = plain.decode(0, kn, vn, lengths, active)
    assert torch.equal(gm, em) and gk.shape == ek.shape == (b, 8, cap, 64)
    for x, y in ((gk, ek), (gv, ev)):
        codes, scales = quant.quantise(y.cpu(), bits)
        assert torch.equal(x.cpu().double(), quant.values(codes, scales, bits))
    with pytest.raises(ValueError, match="exceeds the KV capacity"):
        wide = torch.zeros(b, 8, cap + 1, 64, device=DEV, dtype=BF16)
        cache.prefill(0, slice(0, b), wide, wide, torch.ones(b, cap + 1, device=DEV, dtype=torch.bool))


# --------------------------------------------------------------- attention --

@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("b,hq,hkv,cap,splits", [
    (3, 2, 2, 1, None), (5, 6, 2, 63, 1), (4, 4, 4, 64, 1), (7, 16, 8, 65, 2), (6, 24, 8, 300, 1), (6, 24, 8, 1300, 3),
    (2, 8, 2, 129, 1), (3, 5, 1, 257, 1), (3, 12, 2, 700, 2), (2, 8, 1, 640, 5), (2, 9, 1, 500, 1), (3, 16, 1, 333, 2),
    (2, 22, 2, 4096, None), (1, 24, 8, 4096, 16), (1, 3, 1, 9000, 100)])
@torch.inference_mode()
def test_attention_matches_oracle(bits, b, hq, hkv, cap, splits):
    cache, k, v = random_cache(bits, b, hkv, cap, cap + hq)
    q = (2 * torch.randn(b, hq, 64, generator=gen(b))).to(BF16)
    used = torch.randint(0, cap + 1, (b,), generator=gen(cap), dtype=torch.int32)
    used[0] = cap
    if b > 1:
        used[1] = min(cap, 1)
    if b > 2:
        used[2] = 0
    flash = QuantFlashDecode(b, hkv, hq // hkv, cap, DEV, num_splits=splits, bits=bits)
    got = flash(q.to(DEV)[:, :, None], *cache.layer(0), None, None, 0.125, used=used.to(DEV))[:, :, 0]
    assert torch.isfinite(got).all()
    check(got, q, k[0], v[0], used, 0.125)
    if b > 2:
        assert not bool(got[2].any())
    again = flash(q.to(DEV)[:, :, None], *cache.layer(0), None, None, 0.125, used=used.to(DEV))[:, :, 0]
    assert torch.equal(got, again)


@pytest.mark.parametrize("bits", [4, 8])
@torch.inference_mode()
def test_attention_lengths_bounds_and_strided_queries(bits):
    """used from lengths and active; below zero, past the bound and past the
    capacity; queries as columns of a wider row; fewer rows than planned."""
    hq, hkv, cap, b = 6, 2, 200, 5
    cache, k, v = random_cache(bits, b, hkv, cap, 3)
    wide = vectors((b, hq + 4, 64), 8).to(DEV)
    q = wide[:, 2:2 + hq].unsqueeze(2)
    flash = QuantFlashDecode(7, hkv, 3, cap, DEV, maximum=150, num_splits=2, bits=bits)
    lengths = torch.tensor([62, 999, 0, 149, 10], device=DEV)
    active = torch.tensor([True, False, True, True, True], device=DEV)
    got = flash(q, *cache.layer(0), lengths, active, 0.125)[:, :, 0]
    check(got, q[:, :, 0].cpu(), k[0], v[0], torch.tensor([63, 1, 1, 150, 11]), 0.125)
    used = torch.tensor([-3, 150, 151, 1 << 30, 149], device=DEV)
    got = flash(q, *cache.layer(0), None, None, 0.125, used=used)[:, :, 0]
    check(got, q[:, :, 0].cpu(), k[0], v[0], torch.tensor([0, 150, 150, 150, 149]), 0.125)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("splits,most", [(None, 8300), (7, 8300), (3, 8300), (1000, 8300), (9, 513)])
@torch.inference_mode()
def test_splits_share_each_rows_own_length(bits, splits, most):
    """Rows of every kind of length in one call, at the edges of stages and of
    splits, and the same graph over other lengths; the fused form beside it, its
    new token in the first, a middle or the last split, or behind the row."""
    cap, hq, hkv = 8320, 3, 1
    lengths = torch.tensor([8300, 8192, 4097, 1025, 513, 512, 511, 449, 448, 65, 64, 1, 0], dtype=torch.int32)
    b = lengths.numel()
    cache, k, v = random_cache(bits, b, hkv, cap, 12)
    q = (2 * torch.randn(b, hq, 64, generator=gen(9))).to(BF16)
    flash = QuantFlashDecode(b, hkv, hq, cap, DEV, maximum=most, num_splits=splits, bits=bits)
    used, qd = lengths.to(DEV), q.to(DEV)[:, :, None]

    out = torch.empty_like(qd)

    def step():
        out.copy_(flash(qd, *cache.layer(0), None, None, 0.125, used=used))

    graph = capture_decode(step, lambda: None)
    for turn in range(3):
        now = lengths.roll(turn)
        used.copy_(now)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        check(out[:, :, 0], q, k[0], v[0], now.clamp(max=most), 0.125)
        assert torch.equal(out, flash(qd, *cache.layer(0), None, None, 0.125, used=used))

    caches = [random_cache(bits, b, hkv, cap, 12)[0] for _ in range(2)]
    part, table = fused_inputs(b, hq, hkv, cap, 4)
    for back in (1, 70, 600, -40):
        used.copy_(lengths)
        positions = (lengths.long() - back).to(DEV)
        want = unfused(flash, caches[0], part, table, positions, None, used, hq, hkv)
        got = flash.fused_qkv(part, table, positions, None, *caches[1].layer(0), 0.125, used, hq)
        assert torch.equal(got, want)
        for x, y in zip(caches[0].layer(0), caches[1].layer(0)):
            assert torch.equal(x, y)


@pytest.mark.parametrize("bits", [4, 8])
@torch.inference_mode()
def test_short_rows_are_cut_by_what_runs_at_once(bits):
    """Rows far below the plan's bound: single stages while the grid's workgroups all run at
    once, else pieces of 256 positions or more, a stage for each wave. Which splits of a row
    ran is read off the maxima that they left in the workspace."""
    hkv, hq, cap, splits = 8, 16, 8192, 8
    resident = 256 * (4 if bits == 4 else 2)
    for b in (resident // (hkv * splits), resident // (hkv * splits) + 1):
        lengths = torch.tensor([300, 1, 64, 65, 256, 257, 512, 513, 700, 2048, 2049, 8192, 0])[torch.arange(b) % 13]
        lengths = lengths.tolist()
        cache = QuantKVCache.empty(1, b, hkv, cap, DEV, bits=bits)
        flash = QuantFlashDecode(b, hkv, 2, cap, DEV, num_splits=splits, bits=bits)
        n = b * hq * splits
        maxima = flash.workspace[n * 64 * 4:][:4 * n].view(torch.float32).view(b, hkv, 2, splits)
        maxima.fill_(float("nan"))
        flash(torch.zeros(b, hq, 1, 64, dtype=BF16, device=DEV), *cache.layer(0), None, None, 0.125,
              used=torch.tensor(lengths, device=DEV))
        ran = ~maxima.isnan()
        assert torch.equal(ran, ran[:, :1, :1].expand_as(ran))
        least = 64 if b * hkv * splits <= resident else 256
        for row, used in zip(ran[:, 0, 0].tolist(), lengths):
            chunk = max(least, 64 * -(-used // (64 * splits)))
            pieces = -(-used // chunk)
            assert row == [True] * pieces + [False] * (splits - pieces), (b, used)


@pytest.mark.parametrize("bits", [4, 8])
@torch.inference_mode()
def test_many_short_rows_in_splits_match_oracle(bits):
    """More workgroups than run at once, rows of every length from none to the bound: the
    oracle, the fused form and the cache it leaves."""
    b, hq, hkv, cap, splits = 140, 3, 1, 2400, 8
    cache, k, v = random_cache(bits, b, hkv, cap, 14)
    used = torch.randint(0, 700, (b,), generator=gen(15), dtype=torch.int32)
    used[:8] = torch.tensor([0, 1, 255, 256, 257, 512, 2399, 2400])
    q = (2 * torch.randn(b, hq, 64, generator=gen(16))).to(BF16)
    flash = QuantFlashDecode(b, hkv, hq, cap, DEV, num_splits=splits, bits=bits)
    got = flash(q.to(DEV)[:, :, None], *cache.layer(0), None, None, 0.125, used=used.to(DEV))[:, :, 0]
    check(got, q, k[0], v[0], used, 0.125)
    part, table = fused_inputs(b, hq, hkv, cap, 4)
    other = random_cache(bits, b, hkv, cap, 14)[0]
    for back in (1, 100, -3):
        positions, device_used = (used.long() - back).to(DEV), used.to(DEV)
        want = unfused(flash, cache, part, table, positions, None, device_used, hq, hkv)
        got = flash.fused_qkv(part, table, positions, None, *other.layer(0), 0.125, device_used, hq)
        assert torch.equal(got, want)
        assert all(torch.equal(x, y) for x, y in zip(cache.layer(0), other.layer(0)))


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("hq,splits", [(6, 1), (16, 3), (2, 1)])
@torch.inference_mode()
def test_masked_positions_are_never_seen(bits, hq, splits):
    """Positions past a row's length hold arbitrary bytes, NaN scales among
    them: the results' bits do not change."""
    hkv, cap, b = 2, 333, 6
    cache, k, v = random_cache(bits, b, hkv, cap, 21)
    q = vectors((b, hq, 1, 64), 2).to(DEV)
    used = torch.tensor([1, 64, 65, 127, 200, 0], dtype=torch.int32)
    flash = QuantFlashDecode(b, hkv, hq // hkv, cap, DEV, num_splits=splits, bits=bits)
    before = flash(q, *cache.layer(0), None, None, 0.125, used=used.to(DEV))
    past = (torch.arange(cap)[None] >= used[:, None]).to(DEV)
    for t in (cache.k, cache.v, cache.scales):
        noise = torch.randint(0, 256, t[0].shape, device=DEV, dtype=torch.uint8)
        t[0].copy_(torch.where(past[:, None, :, None], noise, t[0]))
    cache.scales[0].masked_fill_((past & (torch.arange(cap, device=DEV) % 3 == 0))[:, None, :, None], 255)
    after = flash(q, *cache.layer(0), None, None, 0.125, used=used.to(DEV))
    assert torch.equal(before, after) and torch.isfinite(after).all()
    check(after[:, :, 0], q[:, :, 0].cpu(), k[0], v[0], used, 0.125)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("hq,splits", [(6, 1), (6, 3), (16, 1), (32, 1)])
@torch.inference_mode()
def test_nan_positions_reach_their_own_rows_only(bits, hq, splits):
    """A key that stands for NaN makes NaN of its KV head's query heads in its
    row; a value's block, of its 32 channels; nothing else moves a bit."""
    hkv, cap, b = 2, 260, 4
    cache, _, _ = random_cache(bits, b, hkv, cap, 31)
    q = vectors((b, hq, 1, 64), 4).to(DEV)
    used = torch.tensor([260, 100, 130, 7], dtype=torch.int32, device=DEV)
    flash = QuantFlashDecode(b, hkv, hq // hkv, cap, DEV, num_splits=splits, bits=bits)
    clean = flash(q, *cache.layer(0), None, None, 0.125, used=used)
    g = hq // hkv

    def poison(row, head, position, block):
        cache.scales[0, row, head, position, block] = 255
        side = cache.k if block < 2 else cache.v
        half = side.shape[-1] // 2
        side[0, row, head, position, half * (block % 2):half * (block % 2 + 1)] = 0

    poison(0, 1, 200, 1), poison(1, 0, 99, 0), poison(2, 1, 64, 3), poison(3, 0, 0, 2), poison(3, 1, 7, 0)
    got = flash(q, *cache.layer(0), None, None, 0.125, used=used)
    nan = torch.zeros(b, hq, 1, 64, dtype=torch.bool, device=DEV)
    nan[0, g:], nan[1, :g], nan[2, g:, :, 32:], nan[3, :g, :, :32] = True, True, True, True
    assert torch.equal(got.isnan(), nan)
    assert torch.equal(got[~nan], clean[~nan])


@pytest.mark.parametrize("bits", [4, 8])
@torch.inference_mode()
def test_queries_that_are_not_numbers_stay_in_their_head(bits):
    hq, hkv, cap, b = 6, 2, 150, 3
    cache, _, _ = random_cache(bits, b, hkv, cap, 41)
    q = vectors((b, hq, 1, 64), 6).to(DEV)
    used = torch.tensor([150, 70, 3], dtype=torch.int32, device=DEV)
    flash = QuantFlashDecode(b, hkv, 3, cap, DEV, bits=bits)
    clean = flash(q, *cache.layer(0), None, None, 0.125, used=used)
    q[1, 4, 0, 9] = float("nan")
    got = flash(q, *cache.layer(0), None, None, 0.125, used=used)
    assert bool(got[1, 4].isnan().all())
    keep = torch.ones(b, hq, dtype=torch.bool, device=DEV)
    keep[1, 4] = False
    assert torch.equal(got[keep], clean[keep])


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("pattern", ["ramp", "sawtooth", "wide", "falling"])
@pytest.mark.parametrize("splits,hq", [(1, 6), (3, 6), (1, 16), (2, 24)])
@torch.inference_mode()
def test_scores_that_drift(bits, pattern, splits, hq):
    """Scores that move the running maximum many times, by steps below and
    above the slack of 8 (log2 units) before it rescales."""
    hkv, cap, b = 2, 1024, 5
    g = gen(11)
    q = torch.randn(b, hq, 64, generator=g)
    j = torch.arange(cap, dtype=torch.float32)
    t = dict(ramp=0.06 * j - 10, sawtooth=torch.where((j // 16) % 2 == 0, 5.0, 11.0) * (j // 16 % 5) + 0.01 * j,
             wide=20 * torch.randn(cap, generator=g), falling=30 - 0.05 * j)[pattern]
    lead = q[:, ::hq // hkv]
    kx = t[None, None, :, None] * lead[:, :, None, :] / (0.125 * lead.square().sum(-1))[:, :, None, None]
    kx = (kx + 0.05 * torch.randn(b, hkv, cap, 64, generator=g)).to(BF16)
    vx = torch.randn(b, hkv, cap, 64, generator=g).to(BF16)
    q = q.to(BF16)
    cache = QuantKVCache.empty(1, b, hkv, cap, DEV, bits=bits)
    slots, pos = torch.arange(b).repeat_interleave(cap).to(DEV), torch.arange(cap).repeat(b).to(DEV)
    cache.write(0, *(x.to(DEV).transpose(1, 2).reshape(b * cap, hkv, 1, 64) for x in (kx, vx)), pos, None, slots)
    k, v = (x.cpu().double() for x in cache.read(0))
    used = torch.tensor([1024, 1000, 777, 300, 17], dtype=torch.int32)
    flash = QuantFlashDecode(b, hkv, hq // hkv, cap, DEV, num_splits=splits, bits=bits)
    got = flash(q.to(DEV)[:, :, None], *cache.layer(0), None, None, 0.125, used=used.to(DEV))[:, :, 0]
    check(got, q, k, v, used, 0.125)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("hq,splits", [(6, 1), (16, 2), (24, 1)])
@torch.inference_mode()
def test_scores_far_below_zero(bits, hq, splits):
    """Every score of a row the same number near -2^110: the mean of the values.
    One position at half of it: that one's value."""
    b, hkv, cap = 3, 2, 300
    cache = QuantKVCache.empty(1, b, hkv, cap, DEV, bits=bits)
    k = torch.full((b * cap, hkv, 1, 64), 2.0 ** 50, dtype=BF16, device=DEV)
    k.view(b, cap, hkv, 64)[1, 77] /= 2
    v = vectors((b * cap, hkv, 1, 64), 5).to(DEV)
    cache.write(0, k, v, torch.arange(cap, device=DEV).repeat(b), None,
                torch.arange(b, device=DEV).repeat_interleave(cap))
    q = torch.full((b, hq, 1, 64), -2.0 ** 57, dtype=BF16, device=DEV)
    used = torch.tensor([300, 299, 1], dtype=torch.int32, device=DEV)
    flash = QuantFlashDecode(b, hkv, hq // hkv, cap, DEV, num_splits=splits, bits=bits)
    got = flash(q, *cache.layer(0), None, None, 0.125, used=used)[:, :, 0].cpu().double()
    held = cache.read(0)[1].cpu().double()
    want = torch.stack([held[0].mean(1), held[1, :, 77], held[2, :, 0]]).repeat_interleave(hq // hkv, 1)
    # equal probabilities are exactly 1, so the sums' roundings and the result's remain
    tol = 2.0 ** -8 * want.abs() + 2.0 ** -24 * 364 * held.abs().amax()
    assert bool(((got - want).abs() <= tol).all())


def rising_scores(b, hq, hkv, cap, low, step, seed):
    """Queries and keys (bf16) whose scores, scaled by 1/8, rise from ``low`` by ``step`` a
    position for the first query head of each KV head."""
    g = gen(seed)
    q = torch.randn(b, hq, 64, generator=g)
    lead = q[:, ::hq // hkv]
    t = low + step * torch.arange(cap, dtype=torch.float32)
    k = t[None, None, :, None] * lead[:, :, None, :] / (0.125 * lead.square().sum(-1))[:, :, None, None]
    return q.to(BF16), k.to(BF16)


def filled_cache(bits, k, v):
    """A cache of ``k, v [B, Hkv, C, 64]`` (bf16, CPU) and the values it stands for (64 bits, CPU)."""
    b, hkv, cap, _ = k.shape
    cache = QuantKVCache.empty(1, b, hkv, cap, DEV, bits=bits)
    slots, pos = torch.arange(b).repeat_interleave(cap).to(DEV), torch.arange(cap).repeat(b).to(DEV)
    cache.write(0, *(x.to(DEV).transpose(1, 2).reshape(b * cap, hkv, 1, 64) for x in (k, v)), pos, None, slots)
    return cache, *(x.cpu().double() for x in cache.read(0))


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("splits,hq,cap", [(1, 6, 300), (3, 6, 300), (1, 16, 300), (1, 32, 300), (1, 6, 1100)])
@torch.inference_mode()
def test_values_to_the_ends_of_the_range(bits, splits, hq, cap):
    """Values near bf16's largest, of both signs, beside zeros in their block and at other
    positions, under scores that rise by less than the running maximum's slack: finite
    and within the bound. The same with values near 2^-60."""
    hkv, b = 2, 3
    q, k = rising_scores(b, hq, hkv, cap, -4.0, 0.02, 17)
    used = torch.tensor([cap, cap - 1, 70], dtype=torch.int32)
    flash = QuantFlashDecode(b, hkv, hq // hkv, cap, DEV, num_splits=splits, bits=bits)
    for size in (1.6 * 2.0 ** 127, 2.0 ** -60):
        v = size * (1 - 2 * torch.rand(b, hkv, cap, 64, generator=gen(18)))
        j = torch.arange(cap)
        one = torch.nn.functional.one_hot(j % 32, 32)[None, None] * size * (1 - 2 * (j // 5 % 2))[:, None]
        v[..., :32] = torch.where((j % 3 == 0)[:, None], one, torch.zeros(()))
        cache, kd, vd = filled_cache(bits, k, v.to(BF16))
        got = flash(q.to(DEV)[:, :, None], *cache.layer(0), None, None, 0.125, used=used.to(DEV))[:, :, 0]
        assert torch.isfinite(got).all()
        check(got, q, kd, vd, used, 0.125)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("splits,hq,cap", [(1, 6, 300), (3, 6, 300), (1, 16, 300), (1, 6, 1100)])
@pytest.mark.parametrize("power", [123, -100])
@torch.inference_mode()
def test_queries_to_the_ends_of_the_range(bits, splits, hq, cap, power):
    """Queries near bf16's largest over keys as small as they are large, and the reverse:
    ordinary scores, so ordinary results."""
    hkv, b = 2, 3
    q, k = rising_scores(b, hq, hkv, cap, -4.0, 0.02, 19)
    q, k = q * 2.0 ** power, k * 2.0 ** -power
    used = torch.tensor([cap, cap - 1, 70], dtype=torch.int32)
    cache, kd, vd = filled_cache(bits, k, vectors((b, hkv, cap, 64), 20))
    flash = QuantFlashDecode(b, hkv, hq // hkv, cap, DEV, num_splits=splits, bits=bits)
    got = flash(q.to(DEV)[:, :, None], *cache.layer(0), None, None, 0.125, used=used.to(DEV))[:, :, 0]
    assert torch.isfinite(q).all() and torch.isfinite(got).all()
    check(got, q, kd, vd, used, 0.125)


@torch.inference_mode()
def test_attention_past_32_bit_offsets():
    """One KV head whose codes pass 4 GiB: every key zero, so the softmax is
    uniform, and the values that are not zero lie at both ends and around the
    2 and 4 GiB offsets. Sums of 2^26 equal probabilities stay exact in fp32
    (splits of 2^18 positions, powers of two)."""
    cap, used = (1 << 26) + 256, 1 << 26
    cache = QuantKVCache.empty(1, 1, 1, cap, DEV, bits=8)
    positions = torch.tensor([0, (1 << 25) - 1, 1 << 25, used - 1, used, used + 100], device=DEV)
    x = (1 << 20) * torch.ones(6, 1, 1, 64, dtype=BF16, device=DEV)
    x[:, :, :, 32:] *= torch.arange(1, 7, device=DEV)[:, None, None, None]
    zero = torch.zeros(6, dtype=torch.long, device=DEV)
    cache.write(0, torch.zeros_like(x), x, positions, None, zero)
    assert torch.equal(kv_quant.read(cache, 0, positions, zero)[1], x)
    flash = QuantFlashDecode(1, 1, 2, cap, DEV, maximum=used, num_splits=256, bits=8)
    q = torch.randn(1, 2, 1, 64, device=DEV).to(BF16)
    got = flash(q, *cache.layer(0), None, None, 0.125, used=torch.tensor([used], device=DEV))[0, :, 0].float().cpu()
    want = torch.cat((torch.full((32,), 4.0), torch.full((32,), 10.0))) * 2.0 ** -6
    assert torch.equal(got, want.expand(2, 64))


# -------------------------------------------------------------- fused form --

def fused_inputs(b, hq, hkv, cap, seed, splits=3):
    g = gen(seed)
    part = torch.randn(splits, b, (hq + 2 * hkv) * 64, generator=g).to(DEV)
    table = ops.rope_tables(10000.0, 64, cap, BF16)[0].to(DEV)
    return part, table


def unfused(flash, cache, part, table, positions, active, used, hq, hkv):
    """The same step from the separate operators."""
    qkv = part[0].clone()
    for s in range(1, part.shape[0]):
        qkv += part[s]
    qkv = qkv.to(BF16).view(part.shape[1], hq + 2 * hkv, 64)
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    rotary_embedding(positions, q, k, 64, table)
    cache.write(0, k.unsqueeze(2), v.unsqueeze(2), positions, active)
    return flash(q.unsqueeze(2), *cache.layer(0), None, None, 0.125, used=used)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("b,hq,hkv,cap,splits,slices", [
    (5, 6, 2, 200, 1, 3), (5, 6, 2, 700, 3, 1), (4, 2, 2, 130, 1, 2), (6, 16, 8, 257, 2, 8), (6, 24, 8, 300, 1, 4),
    (5, 16, 2, 321, 1, 3), (5, 32, 2, 200, 2, 3), (70, 6, 2, 90, 1, 3)])
@torch.inference_mode()
def test_fused_equals_the_separate_operators(bits, b, hq, hkv, cap, splits, slices):
    """Bit for bit, outputs and cache: an inactive row, positions outside the
    row's length, outside the capacity and below zero, an empty row, at stage
    edges; with a row order and in fragment order."""
    caches = [random_cache(bits, b, hkv, cap, 51)[0] for _ in range(3)]
    part, table = fused_inputs(b, hq, hkv, cap, 5, slices)
    used = torch.randint(1, cap + 1, (b,), generator=gen(6), dtype=torch.int32)
    used[:4] = torch.tensor([cap, 64, 65, 1])
    positions = used.long() - 1
    active = torch.ones(b, dtype=torch.bool)
    if b > 4:
        positions[4], active[0] = used[4].long(), False   # stored past what the row attends
    used, positions, active = used.to(DEV), positions.to(DEV), active.to(DEV)
    flash = QuantFlashDecode(b, hkv, hq // hkv, cap, DEV, num_splits=splits, bits=bits)
    order = torch.argsort(used, descending=True, stable=True).int()
    for step in range(3):
        if step == 1:
            positions = positions.clone()
            positions[0], positions[1], positions[2] = cap, -1, cap + 5
        if step == 2:
            used = used.clone()
            used[:] = 0
            used[1] = 40
        want = unfused(flash, caches[0], part, table, positions, active, used, hq, hkv)
        got = flash.fused_qkv(part, table, positions, active, *caches[1].layer(0), 0.125, used, hq)
        frag = flash.fused_qkv(part, table, positions, active, *caches[2].layer(0), 0.125, used, hq, row_order=order,
                               frag_out=True)
        assert torch.equal(got, want)
        assert torch.equal(frag.to_rows(), want.view(b, -1))
        for other in caches[1:]:
            for x, y in zip(caches[0].layer(0), other.layer(0)):
                assert torch.equal(x, y)
        part = part.roll(1, 1)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("hq,splits", [(6, 1), (6, 3), (16, 1), (32, 1)])
@torch.inference_mode()
def test_fused_over_positions_that_were_never_written(bits, hq, splits):
    """The new token's position and all behind it hold the worst bytes there are,
    8-bit codes that are no numbers and NaN scales: they are replaced or never
    looked at."""
    b, hkv, cap = 7, 2, 333
    used = torch.tensor([1, 2, 64, 65, 100, 129, 333], dtype=torch.int32, device=DEV)
    positions = used.long() - 1
    caches = [random_cache(bits, b, hkv, cap, 55)[0] for _ in range(2)]
    behind = (torch.arange(cap, device=DEV)[None] >= positions[:, None])[:, None, :, None]
    for t, worst in zip(caches[1].layer(0), (0x7f, 0xff, 0xff)):
        t.masked_fill_(behind, worst)
    part, table = fused_inputs(b, hq, hkv, cap, 8)
    flash = QuantFlashDecode(b, hkv, hq // hkv, cap, DEV, num_splits=splits, bits=bits)
    want, got = (flash.fused_qkv(part, table, positions, None, *c.layer(0), 0.125, used, hq) for c in caches)
    assert torch.isfinite(want).all() and torch.equal(got, want)
    at = (torch.arange(b, device=DEV), slice(None), positions)
    assert all(torch.equal(x[at], y[at]) for x, y in zip(caches[0].layer(0), caches[1].layer(0)))
    again = flash(torch.zeros(b, hq, 1, 64, dtype=BF16, device=DEV), *caches[1].layer(0), None, None, 0.125, used=used)
    assert torch.isfinite(again).all()


# Few rows whose splits span 1024 positions or more take workgroups of eight waves in 4
# bits. Groups of 3, 8 and 16 query heads; one split and two.
EIGHT_WAVES = pytest.mark.parametrize("cap,splits", [(1100, 1), (2100, 1), (2100, 2)])
GROUPS = pytest.mark.parametrize("groups", [3, 8, 16])


def eight_wave_lengths(cap):
    """Lengths at the edges of a workgroup's first and second round of stages."""
    return torch.tensor([cap, 1025, 1024, 1023, 513, 512, 511, 449, 65, 64, 1, 0], dtype=torch.int32)


@EIGHT_WAVES
@GROUPS
@torch.inference_mode()
def test_eight_waves_match_oracle(cap, splits, groups):
    hkv, used = 2, eight_wave_lengths(cap)
    b, hq = used.numel(), groups * hkv
    cache, k, v = random_cache(4, b, hkv, cap, 101)
    q = (2 * torch.randn(b, hq, 64, generator=gen(102))).to(BF16)
    flash = QuantFlashDecode(b, hkv, groups, cap, DEV, num_splits=splits, bits=4)
    got = flash(q.to(DEV)[:, :, None], *cache.layer(0), None, None, 0.125, used=used.to(DEV))[:, :, 0]
    check(got, q, k[0], v[0], used, 0.125)
    assert not bool(got[-1].any())


@EIGHT_WAVES
@GROUPS
@torch.inference_mode()
def test_eight_waves_fused_equals_the_separate_operators(cap, splits, groups):
    hkv, used = 2, eight_wave_lengths(cap)
    b, hq = used.numel(), groups * hkv
    caches = [random_cache(4, b, hkv, cap, 103)[0] for _ in range(3)]
    part, table = fused_inputs(b, hq, hkv, cap, 104)
    active = torch.ones(b, dtype=torch.bool, device=DEV)
    active[4] = False
    flash = QuantFlashDecode(b, hkv, groups, cap, DEV, num_splits=splits, bits=4)
    order = torch.arange(b, device=DEV, dtype=torch.int32).flip(0).contiguous()
    for back in (1, 500, -2):
        positions, device_used = (used.long() - back).to(DEV), used.to(DEV)
        want = unfused(flash, caches[0], part, table, positions, active, device_used, hq, hkv)
        got = flash.fused_qkv(part, table, positions, active, *caches[1].layer(0), 0.125, device_used, hq)
        frag = flash.fused_qkv(part, table, positions, active, *caches[2].layer(0), 0.125, device_used, hq,
                               row_order=order, frag_out=True)
        assert torch.equal(got, want) and torch.equal(frag.to_rows(), want.view(b, -1))
        for other in caches[1:]:
            assert all(torch.equal(x, y) for x, y in zip(caches[0].layer(0), other.layer(0)))


@EIGHT_WAVES
@GROUPS
@torch.inference_mode()
def test_eight_waves_see_only_their_rows(cap, splits, groups):
    """Garbage and NaN scales behind the rows' ends move no bit; a key and a value that stand
    for NaN, and a query that is none, make NaN of their own rows and heads only; the new
    token's place may hold anything."""
    hkv, used = 2, eight_wave_lengths(cap)
    b, hq = used.numel(), groups * hkv
    used = used.to(DEV)
    cache, _, _ = random_cache(4, b, hkv, cap, 105)
    q = vectors((b, hq, 1, 64), 106).to(DEV)
    flash = QuantFlashDecode(b, hkv, groups, cap, DEV, num_splits=splits, bits=4)
    clean = flash(q, *cache.layer(0), None, None, 0.125, used=used)
    assert torch.isfinite(clean).all()
    past = (torch.arange(cap, device=DEV)[None] >= used[:, None])[:, None, :, None]
    for t, worst in zip(cache.layer(0), (0xff, 0x7f, 0xff)):
        t.masked_fill_(past, worst)
    assert torch.equal(flash(q, *cache.layer(0), None, None, 0.125, used=used), clean)

    part, table = fused_inputs(b, hq, hkv, cap, 107)
    other = QuantKVCache.over(*(t.clone() for t in (cache.k, cache.v, cache.scales)))
    for t, worst in zip(other.layer(0), (0xff, 0xff, 0xff)):
        t[torch.arange(b - 1), :, (used[:-1] - 1).long()] = worst
    spare = [QuantKVCache.over(*(t.clone() for t in (cache.k, cache.v, cache.scales))), other]
    got = [flash.fused_qkv(part, table, used.long() - 1, None, *c.layer(0), 0.125, used, hq) for c in spare]
    assert torch.isfinite(got[0]).all() and torch.equal(*got)

    nan = torch.zeros(b, hq, 1, 64, dtype=torch.bool, device=DEV)
    for row, head, position, block in ((0, 1, 1023, 1), (1, 0, 1024, 2), (2, 1, 512, 3), (6, 0, 0, 0)):
        cache.scales[0, row, head, position, block] = 255
        side = cache.k if block < 2 else cache.v
        side[0, row, head, position, 16 * (block % 2):16 * (block % 2 + 1)] = 0
        channels = slice(None) if block < 2 else slice(32 * (block - 2), 32 * (block - 1))
        nan[row, groups * head:groups * (head + 1), :, channels] = True
    q[3, hq - 1, 0, 5] = float("nan")
    nan[3, hq - 1] = True
    got = flash(q, *cache.layer(0), None, None, 0.125, used=used)
    assert torch.equal(got.isnan(), nan) and torch.equal(got[~nan], clean[~nan])


@pytest.mark.parametrize("bits", [4, 8])
@torch.inference_mode()
def test_fused_matches_oracle(bits):
    b, hq, hkv, cap = 6, 24, 8, 150
    cache, k, v = random_cache(bits, b, hkv, cap, 61)
    k, v = k[0].clone(), v[0].clone()
    part, table = fused_inputs(b, hq, hkv, cap, 7)
    used = torch.tensor([150, 64, 65, 1, 100, 129], dtype=torch.int32)
    positions = used.long() - 1
    qkv = part.double().sum(0).to(BF16).cpu().view(b, hq + 2 * hkv, 64)
    _, cos, sin = ops.rope_tables(10000.0, 64, cap, BF16)
    rope = lambda x: torch.stack([x[i] * cos[p] + ops.rotate_half(x[i]) * sin[p] for i, p in enumerate(positions)])
    q = rope(qkv[:, :hq])
    for side, x in ((k, rope(qkv[:, hq:hq + hkv])), (v, qkv[:, hq + hkv:])):
        codes, scales = quant.quantise(x, bits)
        side[torch.arange(b), :, positions] = quant.values(codes, scales, bits)
    flash = QuantFlashDecode(b, hkv, 3, cap, DEV, bits=bits)
    got = flash.fused_qkv(part, table, positions.to(DEV), None, *cache.layer(0), 0.125, used.to(DEV), hq)
    for x, y in zip(cache.read(0), (k, v)):
        assert torch.equal(x.cpu().double(), y)
    check(got[:, :, 0], q, k, v, used, 0.125)


@pytest.mark.parametrize("bits", [4, 8])
@torch.inference_mode()
def test_captured_steps_replay(bits):
    """A step recorded once and replayed as lengths grow, with eager work between
    the replays, against the eager calls; a second object's graph beside it."""
    b, hq, hkv, cap = 3, 6, 2, 1100
    part, table = fused_inputs(b, hq, hkv, cap, 9)
    start = torch.tensor([900, 62, 0], device=DEV)
    outs = []
    for which in range(2):
        cache = random_cache(bits, b, hkv, cap, 71)[0]
        flash = QuantFlashDecode(b, hkv, 3, cap, DEV, bits=bits)
        positions, p = start.clone(), part.clone()
        keep = {}

        def step():
            keep["out"] = flash.fused_qkv(p, table, positions, None, *cache.layer(0), 0.125, (positions + 1).int(), hq)
            keep["back"] = kv_quant.read(cache, 0, positions, cache.slots)
            positions.add_(1)

        saved = [t.clone() for t in (cache.k, cache.v, cache.scales)]

        def reset():
            positions.copy_(start)
            for t, s in zip((cache.k, cache.v, cache.scales), saved):
                t.copy_(s)

        graph = capture_decode(step, reset) if which else None
        reset()
        got = []
        for i in range(5):
            p.copy_(part.roll(i, 1))
            graph.replay() if which else step()
            torch.cuda.synchronize()
            got.append([keep["out"].clone(), *(x.clone() for x in keep["back"])])
            torch.randn(1000, device=DEV).sum()
        outs.append((got, [t.clone() for t in (cache.k, cache.v, cache.scales)]))
    for a, c in zip(*(o[0] for o in outs)):
        assert all(torch.equal(x, y) for x, y in zip(a, c))
    assert all(torch.equal(x, y) for x, y in zip(outs[0][1], outs[1][1]))


@torch.inference_mode()
def test_calls_on_another_stream():
    bits, b, hq, hkv, cap = 4, 4, 6, 2, 1500
    cache, k, v = random_cache(bits, b, hkv, cap, 81)
    q = vectors((b, hq, 1, 64), 3).to(DEV)
    used = torch.tensor([1500, 800, 1, 0], dtype=torch.int32, device=DEV)
    planned = [QuantFlashDecode(b, hkv, 3, cap, DEV, num_splits=4, bits=bits) for _ in range(2)]
    want = planned[0](q, *cache.layer(0), None, None, 0.125, used=used)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    results = []
    for _ in range(8):                       # two streams at once, a plan each
        with torch.cuda.stream(side):
            results.append(planned[1](q, *cache.layer(0), None, None, 0.125, used=used))
        results.append(planned[0](q, *cache.layer(0), None, None, 0.125, used=used))
    torch.cuda.synchronize()
    assert all(torch.equal(r, want) for r in results)


@torch.inference_mode()
def test_refusals_on_the_device():
    cache = QuantKVCache.empty(1, 2, 2, 64, DEV, bits=4)
    eight = QuantKVCache.empty(1, 2, 2, 64, DEV, bits=8)
    x = torch.zeros(2, 2, 1, 64, dtype=BF16, device=DEV)
    pos = torch.zeros(2, dtype=torch.long, device=DEV)
    for bad in (x.float(), x[:, :1], x[..., :32], x.cpu()):
        with pytest.raises(ValueError):
            cache.write(0, bad, bad, pos, None)
    with pytest.raises(ValueError, match="one entry per row"):
        cache.write(0, x, x, pos[:1], None)
    with pytest.raises(ValueError, match="one entry per row"):
        cache.write(0, x, x, pos.cpu(), None)
    flash = QuantFlashDecode(2, 2, 1, 64, DEV, bits=4)
    layer = cache.layer(0)
    used = torch.ones(2, dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError, match="another cache type"):
        flash(x, *eight.layer(0), None, None, 0.125, used=used)
    with pytest.raises(ValueError, match="batch/capacity"):
        flash(torch.zeros(3, 2, 1, 64, dtype=BF16, device=DEV), *layer, None, None, 0.125, used=used)
    with pytest.raises(ValueError, match="batch/capacity"):
        flash(x, *QuantKVCache.empty(1, 2, 2, 32, DEV, bits=4).layer(0), None, None, 0.125, used=used)
    with pytest.raises(ValueError, match="Query heads"):
        flash(torch.zeros(2, 4, 1, 64, dtype=BF16, device=DEV), *layer, None, None, 0.125, used=used)
    with pytest.raises(ValueError, match="16-byte aligned"):
        flash(torch.zeros(2, 2, 1, 72, dtype=BF16, device=DEV)[..., 4:68], *layer, None, None, 0.125, used=used)
    with pytest.raises(ValueError, match="one entry per row"):
        flash(x, *layer, None, None, 0.125, used=used[:1])
    part, table = fused_inputs(2, 2, 2, 64, 1)
    with pytest.raises(ValueError, match="do not match"):
        flash.fused_qkv(part[..., :-64], table, pos, None, *layer, 0.125, used, 2)
    with pytest.raises(ValueError, match="cos/sin"):
        flash.fused_qkv(part, table.float(), pos, None, *layer, 0.125, used, 2)
    with pytest.raises(ValueError, match="permutation"):
        flash.fused_qkv(part, table, pos, None, *layer, 0.125, used, 2, row_order=pos)
    assert not any(bool(t.any()) for t in layer)


# -------------------------------------------------- a model on the cache --

def small_model(seed=3, capacity=128, **over):
    cfg = preset("granite-1b", num_hidden_layers=2, vocab_size=512, **over)
    weights = synth.granite_weights(cfg, seed=seed, device=DEV)
    ep = ExpertParallel(1, 0, 4096, cfg.hidden_size, cfg.num_experts_per_tok, BF16, DEV, HipFusedExperts())
    return cfg, Granite(cfg, weights, ep, capacity)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("epilogue", [True, False])
@torch.inference_mode()
def test_prefill_writes_what_the_bf16_cache_holds(bits, epilogue):
    """Packed and padded prefills: the logits are the bf16 cache's, bit for bit
    (prefill attends over its own keys), and the cache is that one's, quantised."""
    cfg, model = small_model()
    model.qkv_epilogue = epilogue
    lengths = [9, 33, 1]
    caches = [KVCache(cfg, 3, 64, DEV, BF16), QuantKVCache(cfg, 3, 64, DEV, BF16, bits=bits)]
    packed, ends = build_packed(lengths, DEV)
    tokens = torch.randint(1, 512, (1, sum(lengths)), generator=gen(1)).to(DEV)
    valid = torch.ones_like(tokens, dtype=torch.bool)
    logits = [model.forward(tokens, packed.positions[None], valid, c, slot=packed, last=ends.long() - 1)
              for c in caches]
    assert torch.equal(*logits)
    padded = torch.randint(1, 512, (2, 20), generator=gen(2)).to(DEV)
    columns = torch.arange(20, device=DEV)[None].expand(2, -1)
    keep = columns < torch.tensor([20, 6], device=DEV)[:, None]
    logits = [model.forward(padded, columns, keep, c, slot=slice(0, 2), last=torch.tensor([19, 5])) for c in caches]
    assert torch.equal(*logits)
    for layer in range(2):
        for got, held in zip(caches[1].read(layer), (caches[0].k[layer], caches[0].v[layer])):
            codes, scales = quant.quantise(held.cpu(), bits)
            assert torch.equal(got.cpu().double(), quant.values(codes, scales, bits))


@pytest.mark.parametrize("bits", [4, 8])
@torch.inference_mode()
def test_decode_layer_is_its_operators(bits):
    """Both decode layers of the model (split-K projections with the fused
    attention, and the dense ones with a store of its own) are bit for bit the
    operators called one by one, an inactive row among them."""
    cfg, model = small_model()
    b, cap, hq, hkv = 5, 64, 16, 8
    caches = [random_cache(bits, b, hkv, cap, 91, layers=2)[0] for _ in range(4)]
    w = model.w["layers"][1]
    z = (vectors((b, cfg.hidden_size), 4)).to(DEV)
    positions = torch.tensor([40, 1, 0, 63, 5], device=DEV)
    active = torch.tensor([True, True, True, True, False], device=DEV)
    model.used = (positions + 1).int()
    splits = model.decode_splits(b)
    got = model.attention_splitk(z, w, caches[0], 1, positions, active, splits)
    flash = QuantFlashDecode(b, hkv, hq // hkv, cap, DEV, bits=bits)
    part = linear_splitk(z, w["self_attn.qkv_proj"], splits[0])
    a = flash.fused_qkv(part, model.cos_sin, positions, active, *caches[1].layer(1), cfg.attention_multiplier,
                        model.used, hq, frag_out=True)
    assert torch.equal(got, linear_splitk_frag(a, w["self_attn.o_proj"], splits[1]))
    for epilogue in (True, False):
        model.qkv_epilogue = epilogue
        got = model.attention(z, w, caches[2], 1, positions, active, positions, None)
        qkv = linear_rope_kv(z, w["self_attn.qkv_proj"], hq, hkv, positions, active, model.cos_sin, None, 1)
        heads = qkv.view(b, hq + 2 * hkv, 1, 64)
        caches[3].write(1, heads[:, hq:hq + hkv], heads[:, hq + hkv:], positions, active)
        a = flash(heads[:, :hq], *caches[3].layer(1), None, None, cfg.attention_multiplier, used=model.used)
        assert torch.equal(got, linear_dense(a.view(b, -1), w["self_attn.o_proj"]))
    for one, two in ((caches[0], caches[1]), (caches[2], caches[3])):
        assert all(torch.equal(x, y) for x, y in zip((one.k, one.v, one.scales), (two.k, two.v, two.scales)))
    fresh = random_cache(bits, b, hkv, cap, 91, layers=2)[0]
    moved = (caches[0].scales != fresh.scales).any(-1) | (caches[0].k != fresh.k).any(-1)
    at = torch.zeros(2, b, 1, cap, dtype=torch.bool, device=DEV)
    at[1, torch.arange(4), 0, positions[:4]] = True
    assert torch.equal(moved & ~at, torch.zeros_like(moved)) and bool((moved & at).any())


@pytest.mark.parametrize("lean", [True, False])
@torch.inference_mode()
def test_decode_forward_runs_on_the_quantised_cache(lean):
    """A whole decode step through ``Granite.forward``, lean and masked: finite
    logits, the new tokens stored, a masked row's cache untouched."""
    cfg, model = small_model()
    model.decode_lean = lean
    cache = random_cache(4, 4, 8, 64, 93, layers=2)[0]
    tokens = torch.randint(1, 512, (4, 1), generator=gen(3)).to(DEV)
    positions = torch.tensor([[40], [1], [0], [63]], device=DEV)
    valid = torch.tensor([[True], [True], [True], [False]], device=DEV)
    before = cache.scales.clone(), cache.k.clone()
    logits = model.forward(tokens, positions, valid, cache)
    assert logits.shape == (4, 1, 512) and torch.isfinite(logits).all()
    moved = (cache.k != before[1]).any(-1).any(0).any(1)
    expected = torch.zeros(4, 64, dtype=torch.bool, device=DEV)
    expected[torch.arange(3), positions[:3, 0]] = True
    assert torch.equal(moved, expected)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("model_name", ["granite-1b", "granite-3b"])
@torch.inference_mode()
def test_engine_runs_on_the_quantised_cache(bits, model_name):
    """Generation over ragged prompts: the captured asynchronous steps and the
    eager ones give the same tokens and the same cache bytes, twice over, and
    the first tokens are the bf16 engine's."""
    cfg = preset(model_name, num_hidden_layers=2, vocab_size=512)
    weights = synth.granite_weights(cfg, seed=5, device=DEV)
    prompts = synth.prompts(5, [40, 3, 17, 64, 1], cfg.vocab_size, 7)
    runs = []
    for mode, kv_bits in (("eager", bits), ("graph-async", bits), ("graph", bits), ("eager", 16)):
        ep = ExpertParallel(1, 0, 4096, cfg.hidden_size, cfg.num_experts_per_tok, BF16, DEV, HipFusedExperts())
        model = Granite(cfg, weights, ep, 128)
        requests = [Request(str(i), p, 12) for i, p in enumerate(prompts)]
        run = OptimizedEngine(model, requests, mode=mode, ignore_eos=True, kv_bits=kv_bits, capacity=128)
        first, _ = run.generate()
        second, _ = run.generate()
        assert first == second and all(len(o) == 12 for o in first.values())
        runs.append((first, [] if kv_bits == 16 else [t.clone() for t in (run.cache.k, run.cache.v, run.cache.scales)]))
    for other in runs[1:3]:
        assert other[0] == runs[0][0]
        assert all(torch.equal(a, c) for a, c in zip(other[1], runs[0][1]))
    assert all(runs[3][0][r][0] == o[0] for r, o in runs[0][0].items())


@pytest.mark.parametrize("kind", [Engine, BatchPrefillEngine])
@torch.inference_mode()
def test_every_engine_takes_the_quantised_cache(kind):
    """The engines without the optimized policy (masked decode, one padded
    prefill per request or per batch): eager and captured steps agree, and the
    first tokens are the bf16 cache's."""
    cfg, _ = small_model()
    prompts = synth.prompts(3, [5, 21, 9], cfg.vocab_size, 7)
    runs = []
    for mode, kv_bits in (("eager", 8), ("graph", 8), ("eager", 16)):
        model = small_model()[1]
        run = kind(model, [Request(str(i), p, 6) for i, p in enumerate(prompts)], mode=mode, ignore_eos=True,
                   kv_bits=kv_bits, capacity=64)
        out, _ = run.generate()
        assert all(len(o) == 6 for o in out.values())
        runs.append((out, run.cache.k.clone()))
    assert runs[0][0] == runs[1][0] and torch.equal(runs[0][1], runs[1][1])
    assert all(runs[2][0][r][0] == o[0] for r, o in runs[0][0].items())


@torch.inference_mode()
def test_decode_attention_of_the_other_cache_is_refused():
    cfg, model = small_model()
    cache = QuantKVCache(cfg, 2, 64, DEV, BF16)
    model.decode_flash = FlashDecode(2, 8, 2, 64, DEV)
    tokens, positions = torch.ones(2, 1, dtype=torch.long, device=DEV), torch.zeros(2, 1, dtype=torch.long, device=DEV)
    with pytest.raises(ValueError, match="another KV cache type"):
        model.forward(tokens, positions, torch.ones(2, 1, dtype=torch.bool, device=DEV), cache)
