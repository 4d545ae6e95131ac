"""The paged KV cache on the GPU: rotary store, read-back, decode attention, weights
and eviction against the oracle in 64 bits (oracle/paged.py).

Copies, indices and the bf16 table's arithmetic are exact. The other tolerances are
derived (:func:`rotated_bound`, :func:`attention_bound`, :func:`weight_bound`).
"""
import math

import pytest
import torch

from litemoe_amd import kv_paged, rope, synth
from litemoe_amd._lib import NativeError
from litemoe_amd.batch import BatchPrefillEngine, prefill_logits
from litemoe_amd.cache import KVCache, PagedKVCache, QuantKVCache
from litemoe_amd.config import preset
from litemoe_amd.engine import Engine, Request
from litemoe_amd.ep import ExpertParallel
from litemoe_amd.experts import HipFusedExperts
from litemoe_amd.flash_decode import FlashDecode, PagedFlashDecode, QuantFlashDecode
from litemoe_amd.linear import linear_dense, linear_rope_kv, linear_splitk, linear_splitk_frag
from litemoe_amd.model import Granite
from litemoe_amd.optimized import OptimizedEngine
from litemoe_amd.packed import build_packed, packed_prefill_logits
from oracle import paged

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16


def gen(seed):
    return torch.Generator().manual_seed(seed)


def vectors(shape, seed):
    """bf16 vectors whose channels have unequal sizes."""
    g = gen(seed)
    return (torch.randn(shape, generator=g) * torch.exp(0.5 * torch.randn(shape[-1], generator=g))).to(BF16)


def random_cache(lengths, heads, dim, page, seed, layers=1, capacity=None, junk=math.nan, hole=False):
    """A cache whose rows hold ``lengths`` positions in pages of no order, everything else ``junk``, and the
    rest of the table out of range. ``hole``: a page in the middle of the longest row is missing."""
    need = [-(-n // page) for n in lengths]
    width = max(1, *need) if capacity is None else -(-capacity // page)
    pages = sum(need) + 3
    ids = torch.randperm(pages, generator=gen(seed)).tolist()
    table = torch.tensor([-1, pages, -(2 ** 31), 2 ** 31 - 1], dtype=torch.int32).repeat(len(lengths), width)[:, :width]
    table = table.contiguous()
    k, v = (torch.full((layers, pages, heads, page, dim), junk).to(BF16) for _ in range(2))
    for b, n in enumerate(lengths):
        for i in range(need[b]):
            at, count = ids.pop(), min(page, n - i * page)
            table[b, i] = at
            for side, s in ((k, 1), (v, 2)):
                side[:, at, :, :count] = vectors((layers, heads, count, dim), 97 * seed + 13 * b + 5 * i + s)
    if hole:
        b = max(range(len(lengths)), key=lambda i: lengths[i])
        table[b, need[b] // 2] = -7
    cache = PagedKVCache.over(k.to(DEV), v.to(DEV), table.to(DEV))
    return cache, k, v, table


def rotated_bound(x, exact, size=1.0):
    """A rotated value: rounded once to bf16 (2^-8 of it) after two products, a sum and the angles' rounding to
    fp32, each within 2^-24 of |x1 c| + |x2 s| <= 2 size max|x|, five of them."""
    return 2.0 ** -8 * exact.abs() + 5 * 2.0 ** -24 * 2 * size * x.double().abs().amax(-1, keepdim=True) + 1e-38


def attention_bound(q, pk, pv, table, used, scale, out, limit=None):
    """How far outputs may be off, per element, with A = sum p|v| / sum p, n the row's positions:
    * a probability enters the product as two bf16 parts, its first 8 bits (less than 2^-7 of it lost) and the rest,
      rounded (2^-8 of that) and 2^-18 of the whole larger: 2^-15 A + 2^-18 A; the result's own rounding adds 2^-8 of
      it (2^-8 (1 + 2^-6) |out| with what the others move it by);
    * a score's D products are summed in fp32 (D roundings of at most 2^-24 of S = scale sum|q k|), scaled (one of
      the score, one of the scale), and its distance to the reference, at most 2 S + 6, is rounded: (D + 8) S + 8 in
      units of 2^-24; that moves p by the same share, in numerator and denominator;
    * sums over the positions in any order, the exponential and the merges: (n + 64) 2^-24 of A + |out|."""
    b, hq, d = q.shape
    hkv = pk.shape[1]
    tol = torch.zeros(out.shape, dtype=torch.float64)
    for i in range(b):
        n = int(used[i]) if limit is None else min(int(used[i]), limit)
        k, there = paged.row(pk, table, i, n)
        v, _ = paged.row(pv, table, i, n)
        k, v, n = k[:, there], v[:, there], int(there.sum())
        if not n:
            continue
        qi = q[i].double().view(hkv, hq // hkv, d)
        p = torch.softmax(qi @ k.transpose(1, 2) * scale, -1)
        a = (p @ v.abs()).reshape(hq, d)
        size = (qi.abs() @ k.abs().transpose(1, 2)).amax(-1).reshape(hq, 1) * scale
        o = out[i].abs()
        tol[i] = 2.0 ** -8 * (1 + 2.0 ** -6) * o + 1.125 * 2.0 ** -15 * a + 2.0 ** -24 * (2 * ((d + 8) * size + 8) + n + 64) * (a + o)
    return tol + 1e-30


def weight_bound(q, pk, table, b, n, scale, p, before):
    """A position's weight: every probability is off by what :func:`attention_bound` says of p (no rounding to
    bf16 enters here), and the sum over G heads and what was there by a rounding each."""
    hkv, groups, _ = p.shape
    k, there = paged.row(pk, table, b, n)
    qi = q[b].double().view(hkv, groups, -1)
    size = (qi.abs() @ k.abs().transpose(1, 2)).amax(-1).amax(-1)[:, None] * scale
    share = 2 * ((q.shape[2] + 8) * size + 8) + k.shape[1] + 64
    total = p.sum(1)
    return 2.0 ** -24 * ((share + groups + 1) * total + (groups + 1) * before.double().abs()) + 1e-38


def check_attention(got, q, k, v, table, used, scale, limit=None):
    exp, p = paged.attention(q, k, v, table, used, scale, limit)
    got = got.double().cpu().reshape(exp.shape)
    assert torch.isfinite(got).all()
    over = ((got - exp).abs() - attention_bound(q, k, v, table, used, scale, exp, limit)).amax()
    assert float(over) <= 0, float(over)
    return p


# ---------------------------------------------------------- rotation, store --

STORES = [
    # tokens, q heads, kv heads, dim, rotary, page
    (1, 1, 1, 64, 64, 16), (5, 4, 2, 64, 32, 16), (33, 24, 8, 64, 64, 64), (64, 16, 8, 64, 48, 32),
    (7, 8, 1, 128, 128, 128), (130, 3, 3, 128, 64, 16), (300, 16, 8, 64, 16, 256),
]


@pytest.mark.parametrize("f32", [True, False])
@pytest.mark.parametrize("neox", [True, False])
@pytest.mark.parametrize("tokens,hq,hkv,dim,rotary,page", STORES)
@torch.inference_mode()
def test_rotate_and_store(tokens, hq, hkv, dim, rotary, page, neox, f32):
    """Strided heads of a packed projection; positions past the table, rows and positions out of range, inactive
    rows, positions without a page; every cell that no token names stays as it was."""
    batch, capacity, table_len = 3, 2 * max(page, tokens), 400
    cache, *_ = random_cache([capacity] * batch, hkv, dim, page, tokens, layers=2, junk=7.0)
    table = cache.table.cpu()
    table[1, 0] = -1
    cache.table.copy_(table)
    qkv = vectors((tokens, hq + 2 * hkv, dim), tokens).to(DEV)
    q, k, v = qkv.split((hq, hkv, hkv), 1)
    at = torch.randperm(batch * capacity, generator=gen(tokens + 1))[:tokens]
    slots, at = at // capacity, at % capacity
    positions = torch.randint(0, table_len, (tokens,), generator=gen(5))
    active = torch.ones(tokens, dtype=torch.bool)
    if tokens > 4:
        positions[0], positions[1] = table_len, -3
        at[2], at[3], slots[4] = capacity, -1, batch
        active[3::5] = False
    cos, sin = paged.angles(positions.clamp(0, table_len - 1), rotary, 10000.0)
    cos_sin = rope.rotary_table(table_len, rotary, 10000.0, device=DEV, dtype=torch.float32 if f32 else BF16)
    if not f32:
        held = cos_sin.cpu().double()[positions.clamp(0, table_len - 1)]
        cos, sin = held[:, :rotary // 2], held[:, rotary // 2:]
    turned = (positions >= 0) & (positions < table_len)
    before = cache.k.cpu(), cache.v.cpu()
    q_out, k_out = rope.rotate_kv_write(q, k, v, positions.to(DEV), active.to(DEV), cos_sin, cache, 1, slots.to(DEV),
                                        at=at.to(DEV), is_neox=neox, keep_k=True)
    for got, x in ((q_out.cpu(), q.cpu()), (k_out.cpu(), k.cpu())):
        exp = torch.where(turned[:, None, None], paged.rotate(x, cos, sin, neox, rounded=not f32), x.double())
        if f32:
            assert bool(((got.double() - exp).abs() <= rotated_bound(x, exp)).all())
            assert torch.equal(got[..., rotary:], x[..., rotary:]) and torch.equal(got[~turned], x[~turned])
        else:
            assert torch.equal(got, exp.to(BF16))
    expected = [t.clone() for t in before]
    for t in range(tokens):
        c = paged.cell(table, cache.k.shape[1], page, int(slots[t]), int(at[t]))
        if c and active[t]:
            expected[0][1, c[0], :, c[1]] = k_out[t].cpu()
            expected[1][1, c[0], :, c[1]] = v[t].cpu()
    assert torch.equal(cache.k.cpu(), expected[0]) and torch.equal(cache.v.cpu(), expected[1])
    # read-back: what stands there, zeros where nothing can
    back = kv_paged.read(cache, 1, at.to(DEV), slots.to(DEV))
    for got, held in zip(back, expected):
        for t in range(tokens):
            c = paged.cell(table, cache.k.shape[1], page, int(slots[t]), int(at[t]))
            want = held[1, c[0], :, c[1]] if c else torch.zeros(hkv, dim, dtype=BF16)
            assert torch.equal(got[t, :, 0].cpu(), want)
    # the store alone, from any strides, is the same copy
    cache.k.copy_(before[0])
    cache.v.copy_(before[1])
    odd = torch.empty(tokens, hkv, dim + 1, dtype=BF16, device=DEV)[..., 1:]
    odd.copy_(k_out)
    cache.write(1, odd[:, :, None], v[:, :, None], at.to(DEV), active.to(DEV), slots.to(DEV))
    assert torch.equal(cache.k.cpu(), expected[0]) and torch.equal(cache.v.cpu(), expected[1])


@pytest.mark.parametrize("layout", ["bytes", "strided", "int64"])
@torch.inference_mode()
def test_store_by_a_converted_mask(layout):
    """A mask that is converted, with keys and values that have to be copied, in blocks of one size (512 bytes): the
    rows that it names are stored, and no others."""
    tokens, hkv, dim = 4, 1, 64
    cache = PagedKVCache.empty(1, 1, hkv, dim, tokens, DEV, page=16)
    cache.reserve(0, tokens)
    odd = vectors((2, tokens, hkv, 1, dim + 1), 3).to(DEV)[..., 1:]
    mask = torch.tensor([True, False, True, False])
    active = {"bytes": mask.to(torch.uint8).to(DEV), "int64": mask.long().to(DEV),
              "strided": torch.stack((mask, ~mask), 1).to(DEV)[:, 0]}[layout]
    cache.write(0, odd[0], odd[1], torch.arange(tokens, device=DEV), active,
                torch.zeros(tokens, dtype=torch.int64, device=DEV))
    for got, x in zip(cache.read(0), odd.cpu()):
        exp = torch.where(mask[:, None], x[:, 0, 0], torch.zeros((), dtype=BF16))
        assert torch.equal(got[0, 0, :tokens].cpu(), exp) and not got[0, 0, tokens:].any()


@torch.inference_mode()
def test_bf16_table_is_the_contiguous_path():
    """With the reference's table the store is rope_kv_write bit for bit, in place too."""
    tokens, hq, hkv, page = 70, 24, 8, 32
    cos_sin = rope.rotary_table(128, 64, 10000.0, device=DEV, dtype=BF16)
    qkv = vectors((tokens, hq + 2 * hkv, 64), 3).to(DEV)
    q, k, v = (x.clone() for x in qkv.split((hq, hkv, hkv), 1))
    pos = torch.arange(tokens, device=DEV)
    slots, active = torch.zeros(tokens, dtype=torch.int64, device=DEV), torch.ones(tokens, dtype=torch.bool, device=DEV)
    cfg = preset("granite-3b", num_hidden_layers=1)
    plain = KVCache(cfg, 1, 96, DEV, BF16)
    cache = PagedKVCache(cfg, 1, 96, DEV, BF16, page=page)
    cache.reserve(0, tokens)
    q_out, k_out = rope.rotate_kv_write(q, k, v, pos, active, cos_sin, cache, 0, slots, keep_k=True)
    rope.rope_kv_write(q, k, v, pos, active, cos_sin, plain, 0, slots=slots, write_k=True)
    assert torch.equal(q_out, q) and torch.equal(k_out, k)
    assert torch.equal(cache.read(0)[0][:, :, :96], plain.k[0]) and torch.equal(cache.read(0)[1], plain.v[0])


@pytest.mark.parametrize("dim,rotary,neox,f32", [(80, 32, True, True), (256, 256, False, True), (64, 64, False, False),
                                                 (96, 96, True, False), (64, 64, True, True)])
@torch.inference_mode()
def test_rotary_embedding_in_place(dim, rotary, neox, f32):
    tokens = 37
    q, k = vectors((tokens, 5, dim), 1).to(DEV), vectors((tokens, 2, dim), 2).to(DEV)
    positions = torch.randint(0, 90, (tokens,), generator=gen(9))
    cos_sin = rope.rotary_table(90, rotary, 500.0, device=DEV, dtype=torch.float32 if f32 else BF16)
    held = cos_sin.cpu().double()[positions]
    before = q.cpu(), k.cpu()
    rope.rotary_embedding(positions.to(DEV), q, k, dim, cos_sin, is_neox=neox)
    for got, x in zip((q.cpu(), k.cpu()), before):
        exp = paged.rotate(x, held[:, :rotary // 2], held[:, rotary // 2:], neox, rounded=not f32)
        if f32:
            assert bool(((got.double() - exp).abs() <= rotated_bound(x, exp)).all())
        else:
            assert torch.equal(got, exp.to(BF16))


@pytest.mark.parametrize("f32", [True, False])
@pytest.mark.parametrize("layout", ["columns", "in turn", "heads outside"])
@torch.inference_mode()
def test_rotary_embedding_in_place_of_packed_heads(layout, f32):
    """Queries and keys that lie between each other are turned as those that stand alone, and what lies between them
    stays."""
    tokens, heads, dim = 37, 4, 64
    x = vectors({"columns": (tokens, 3 * heads, dim), "in turn": (tokens, heads, 3, dim),
                 "heads outside": (3 * heads, tokens, dim)}[layout], 1).to(DEV)
    before = x.clone()
    parts = {"columns": lambda t: t.split(heads, 1), "in turn": lambda t: t.unbind(2),
             "heads outside": lambda t: t.transpose(0, 1).split(heads, 1)}[layout]
    cos_sin = rope.rotary_table(90, 64, 500.0, device=DEV, dtype=torch.float32 if f32 else BF16)
    positions = torch.randint(0, 90, (tokens,), generator=gen(9)).to(DEV)
    (q, k, v), (q0, k0, v0) = parts(x), parts(before)
    alone = q0.contiguous(), k0.contiguous()
    rope.rotary_embedding(positions, *alone, dim, cos_sin)
    rope.rotary_embedding(positions, q, k, dim, cos_sin)
    assert torch.equal(q, alone[0]) and torch.equal(k, alone[1]) and torch.equal(v, v0)


# --------------------------------------------------------------- attention --

ATTENTIONS = [
    # lengths, kv heads, groups, dim, page, splits
    ([1], 1, 1, 64, 16, None), ([0], 2, 3, 64, 16, None), ([0, 1, 2, 15, 16, 17, 31, 32, 33], 2, 3, 64, 16, None),
    ([509], 8, 2, 64, 16, None), ([509], 8, 2, 64, 16, 1), ([1000, 3, 0, 127, 128, 129], 2, 3, 64, 64, 7),
    ([300, 5], 1, 16, 64, 32, None), ([300, 5], 1, 16, 64, 32, 3), ([95, 96, 97, 64], 3, 8, 64, 128, 2),
    ([1, 0, 33], 1, 1, 128, 16, None), ([700, 40, 0], 2, 4, 128, 256, None), ([513, 16, 31], 2, 5, 128, 32, 4),
    ([260], 1, 16, 128, 64, 1), ([2049, 4001], 2, 2, 64, 32, 16), ([2049, 1500], 1, 6, 64, 64, 40),
    # one split, scores past what a workgroup keeps (8 and 4 tiles stored together)
    ([7800, 100], 1, 4, 64, 16, 1), ([10500, 1], 1, 3, 64, 64, 1), ([4000, 31, 257], 1, 8, 64, 64, 1),
    ([2000, 129], 1, 16, 64, 64, 1), ([3500, 95, 0], 1, 9, 128, 32, 1),
    # and the most it keeps
    ([1920, 60], 1, 16, 128, 128, 1), ([3800, 10], 1, 8, 64, 64, 1), ([4500, 100], 1, 2, 64, 16, 1), ([2900, 31, 257], 1, 3, 128, 64, 1), ([2000, 1], 1, 5, 64, 64, 1),
    ([1100, 40, 0], 2, 8, 64, 32, 1), ([1000, 95], 1, 9, 128, 32, 1), ([600, 129], 1, 16, 64, 64, 1),
    ([512, 480], 1, 16, 128, 64, 1),
]


@pytest.mark.parametrize("hole", [False, True])
@pytest.mark.parametrize("lengths,hkv,groups,dim,page,splits", ATTENTIONS)
@torch.inference_mode()
def test_attention(lengths, hkv, groups, dim, page, splits, hole):
    """NaN in every place that is not a row's, table entries out of range, and (hole) a page missing."""
    seed = sum(lengths) + dim + groups
    cache, k, v, table = random_cache(lengths, hkv, dim, page, seed, hole=hole)
    b, hq = len(lengths), hkv * groups
    q = vectors((b, hq, dim), seed + 1)
    flash = PagedFlashDecode(b, hkv, groups, cache.capacity, DEV, num_splits=splits, head_dim=dim)
    used = torch.tensor(lengths, dtype=torch.int32)
    args = (None, None, dim ** -0.5)
    got = flash(q.to(DEV)[:, :, None], *cache.layer(0), *args, used=used.to(DEV))
    p = check_attention(got, q, k[0], v[0], table, used, dim ** -0.5)
    # the same with weights, out of place and in place, and from strided queries
    wide = torch.full((b, hq, 1, dim + 8), math.nan, dtype=BF16, device=DEV)
    wide[..., :dim] = q.to(DEV)[:, :, None]
    before = torch.rand(b, hkv, cache.capacity, generator=gen(seed))
    w_in, w_out = before.to(DEV), torch.full((b, hkv, cache.capacity), -5.0, device=DEV)
    again = flash(wide[..., :dim], *cache.layer(0), *args, used=used.to(DEV), weights=w_in, weights_out=w_out)
    assert torch.equal(again, got) and torch.equal(w_in.cpu(), before)
    for i, n in enumerate(lengths):
        w = w_out[i].double().cpu()
        assert bool((w[:, n:] == -5.0).all())
        if n:
            exp = before[i, :, :n].double() + p[i].sum(1)
            tol = weight_bound(q, k[0], table, i, n, dim ** -0.5, p[i], before[i, :, :n])
            assert bool(((w[:, :n] - exp).abs() <= tol).all())
    flash(wide[..., :dim], *cache.layer(0), *args, used=used.to(DEV), weights=w_in)
    for i, n in enumerate(lengths):
        assert torch.equal(w_in[i, :, :n], w_out[i, :, :n]) and torch.equal(w_in[i, :, n:].cpu(), before[i, :, n:])


SHARES = [
    # lengths, kv heads, groups, dim, page, shares: more than there are tiles, one, ends inside rows, rows over many
    ([700, 40, 0], 2, 4, 128, 256, 18), ([0, 0], 2, 3, 64, 16, 7), ([1], 1, 1, 64, 16, 5), ([33, 0, 1, 64], 2, 3, 64, 16, 1),
    ([2000, 5, 1, 0, 900], 2, 2, 64, 64, 9), ([509] * 3, 8, 2, 64, 16, 4), ([128, 128, 256, 128], 1, 16, 64, 32, 5),
    ([1500], 2, 9, 128, 32, 40), ([3000, 1], 1, 5, 64, 64, 23), ([*range(0, 130, 2)], 1, 2, 64, 16, 10),
    ([(37 * i) % 211 for i in range(150)], 2, 3, 64, 16, 64), ([0] * 70 + [300] + [0] * 70, 1, 4, 64, 32, 3),
]


@pytest.mark.parametrize("lengths,hkv,groups,dim,page,shares", SHARES)
@torch.inference_mode()
def test_attention_in_shares(lengths, hkv, groups, dim, page, shares):
    """The rows' tiles cut evenly, whatever the rows: outputs, and weights of calls in shares. Twice, bit for bit."""
    seed = sum(lengths) + dim + shares
    cache, k, v, table = random_cache(lengths, hkv, dim, page, seed, hole=len(lengths) == 5)
    b, hq, scale = len(lengths), hkv * groups, dim ** -0.5
    q = vectors((b, hq, dim), seed + 1)
    flash = PagedFlashDecode(b, hkv, groups, cache.capacity, DEV, head_dim=dim)
    flash.splits, flash.shares = 1, shares
    flash.workspace = flash._space(False)
    used = torch.tensor(lengths, dtype=torch.int32)
    args = (q.to(DEV)[:, :, None], *cache.layer(0), None, None, scale, used.to(DEV))
    flash.workspace.fill_(255)
    got = flash(*args)
    p = check_attention(got, q, k[0], v[0], table, used, scale)
    before = torch.rand(b, hkv, cache.capacity, generator=gen(seed))
    w = before.to(DEV)
    flash.weigh_space, flash.weigh_cut = flash._space(True).fill_(255), (1, shares)
    assert torch.equal(flash(*args, weights=w), got)
    for i, n in enumerate(lengths):
        assert torch.equal(w[i, :, n:].cpu(), before[i, :, n:])
        if n:
            tol = weight_bound(q, k[0], table, i, n, scale, p[i], before[i, :, :n])
            assert bool(((w[i, :, :n].double().cpu() - before[i, :, :n].double() - p[i].sum(1)).abs() <= tol).all())
    again = flash(*args)
    assert torch.equal(again, got)


@torch.inference_mode()
def test_shares_are_the_plan_of_large_batches():
    """The plan takes shares where the caller asks for no splits, and their calls agree with the splits'."""
    b, hkv, page, longest = 20, 8, 64, 4000
    assert PagedFlashDecode(b, hkv, 2, 4032, DEV).shares == 0
    b = 40
    lengths = [1 + (1237 * i) % longest for i in range(b)]
    cache, k, v, table = random_cache(lengths, hkv, 64, page, 3, capacity=4032)
    flash = PagedFlashDecode(b, hkv, 2, cache.capacity, DEV)
    split = PagedFlashDecode(b, hkv, 2, cache.capacity, DEV, num_splits=2)
    assert flash.shares == 64 and split.shares == 0 and split.splits == 2
    q = vectors((b, 16, 64), 4)
    used = torch.tensor(lengths, dtype=torch.int32)
    for f in (flash, split):
        got = f(q.to(DEV)[:, :, None], *cache.layer(0), None, None, 0.125, used=used.to(DEV))
        p = check_attention(got, q, k[0], v[0], table, used, 0.125)
        w = torch.zeros(b, hkv, cache.capacity, device=DEV)
        f(q.to(DEV)[:, :, None], *cache.layer(0), None, None, 0.125, used=used.to(DEV), weights=w)
        for i, n in enumerate(lengths):
            tol = weight_bound(q, k[0], table, i, n, 0.125, p[i], torch.zeros(1))
            assert bool(((w[i, :, :n].double().cpu() - p[i].sum(1)).abs() <= tol).all()) and not w[i, :, n:].any()
    # with weights a workgroup keeps the rows' scores, where they fit; else the shares stand
    assert flash.weigh_cut == (1, 0) and split.weigh_cut == (2, 0)
    wide = PagedFlashDecode(b, hkv, 8, cache.capacity, DEV)
    wide._weights(w, w, b, w.get_device())
    assert wide.weigh_cut == (1, 64)


@torch.inference_mode()
def test_used_is_held_to_the_plan_and_the_table():
    lengths = [96, 64, 80]
    cache, k, v, table = random_cache(lengths, 2, 64, 32, 5)
    q = vectors((3, 4, 64), 8)
    flash = PagedFlashDecode(3, 2, 2, cache.capacity, DEV, maximum=70)
    used = torch.tensor([2 ** 31 - 1, -4, 80], dtype=torch.int32)
    got = flash(q.to(DEV)[:, :, None], *cache.layer(0), None, None, 0.125, used=used.to(DEV))
    check_attention(got, q, k[0], v[0], table, used, 0.125, limit=70)
    assert not got[1].any()
    whole = PagedFlashDecode(3, 2, 2, cache.capacity, DEV)
    used = torch.tensor([2 ** 31 - 1, -4, 80], dtype=torch.int32)
    got = whole(q.to(DEV)[:, :, None], *cache.layer(0), None, None, 0.125, used=used.to(DEV))
    check_attention(got, q, k[0], v[0], table, used, 0.125)
    # a row of which no page exists
    cache.table.fill_(-1)
    w = torch.ones(3, 2, cache.capacity, device=DEV)
    got = whole(q.to(DEV)[:, :, None], *cache.layer(0), None, None, 0.125, used=used.to(DEV), weights=w)
    assert not got.any() and bool((w == 1).all())


@pytest.mark.parametrize("value", [math.inf, math.nan, 3.0e38])
@torch.inference_mode()
def test_attended_infinities_stay_in_their_row_and_head(value):
    """An attended V of infinity or NaN, or the type's largest values, reach the channels that hold them, and no
    other row, KV head or channel."""
    cache, k, v, table = random_cache([70, 40], 2, 64, 16, 5)
    q = vectors((2, 4, 64), 8)
    flash = PagedFlashDecode(2, 2, 2, cache.capacity, DEV)
    used = torch.tensor([70, 40], dtype=torch.int32).to(DEV)
    clean = flash(q.to(DEV)[:, :, None], *cache.layer(0), None, None, 0.125, used=used)
    page, place = paged.cell(table, k.shape[1], 16, 0, 37)
    cache.v[0, page, 1, place, 5] = value
    got = flash(q.to(DEV)[:, :, None], *cache.layer(0), None, None, 0.125, used=used)
    same = torch.ones(2, 4, 1, 64, dtype=torch.bool, device=DEV)
    same[0, 2:, 0, 5] = False
    assert torch.equal(got[same], clean[same])
    hit = got[0, 2:, 0, 5].float()
    assert bool((hit.isnan() if math.isnan(value) else hit > 1e30).all())


@torch.inference_mode()
def test_large_scores():
    """Scores far apart: the running maximum moves, in later tiles too."""
    cache, k, v, table = random_cache([400, 200], 1, 64, 16, 3)
    for b, at in ((0, 399), (0, 40), (1, 199), (1, 0)):
        page, place = paged.cell(table, k.shape[1], 16, b, at)
        for pool in (k, cache.k):
            pool[0, page, 0, place] *= 40
    q = vectors((2, 3, 64), 4) * 8
    flash = PagedFlashDecode(2, 1, 3, cache.capacity, DEV, num_splits=2)
    used = torch.tensor([400, 200], dtype=torch.int32)
    got = flash(q.to(DEV)[:, :, None], *cache.layer(0), None, None, 0.125, used=used.to(DEV))
    check_attention(got, q, k[0], v[0], table, used, 0.125)


@torch.inference_mode()
def test_pages_past_32_bits():
    """A pool of more than 2^32 bytes and 2^31 elements a side: the last pages are reached."""
    page, heads = 256, 8
    pages = (2 ** 31) // (heads * page * 64) + 40
    k = torch.empty(1, pages, heads, page, 64, dtype=BF16, device=DEV)
    v = torch.empty_like(k)
    n = 300
    table = torch.tensor([[pages - 1, pages - 2]], dtype=torch.int32, device=DEV)
    cache = PagedKVCache.over(k, v, table)
    q, kn, vn = vectors((1, 16, 64), 1), vectors((n, heads, 64), 2), vectors((n, heads, 64), 3)
    cache.write(0, kn.to(DEV)[:, :, None], vn.to(DEV)[:, :, None], torch.arange(n, device=DEV), None,
                torch.zeros(n, dtype=torch.int64, device=DEV))
    small_k, small_v = (torch.zeros(2, heads, page, 64, dtype=BF16) for _ in range(2))
    for small, x in ((small_k, kn), (small_v, vn)):
        small[0] = x[:page].transpose(0, 1)
        small[1, :, :n - page] = x[page:].transpose(0, 1)
    flash = PagedFlashDecode(1, heads, 2, 512, DEV)
    used = torch.tensor([n], dtype=torch.int32)
    got = flash(q.to(DEV)[:, :, None], *cache.layer(0), None, None, 0.125, used=used.to(DEV))
    check_attention(got, q, small_k, small_v, torch.tensor([[0, 1]], dtype=torch.int32), used, 0.125)


# ------------------------------------------------------------------- fused --

@pytest.mark.parametrize("weighed", [False, True])
@pytest.mark.parametrize("neox,f32,rotary", [(True, False, 64), (True, True, 64), (False, True, 32), (False, False, 48)])
@pytest.mark.parametrize("lengths,hkv,groups,dim,page,splits", [
    ([1], 1, 1, 64, 16, None), ([17, 32, 33, 1, 64], 2, 3, 64, 16, None), ([1000, 500, 31], 8, 2, 64, 64, 4),
    ([130, 129, 128], 1, 16, 64, 128, 2), ([40, 257], 2, 4, 128, 32, None), ([600, 20], 1, 16, 128, 256, 3),
    ([1100, 40, 97], 2, 8, 64, 32, 1), ([1000, 95], 1, 9, 128, 32, 1), ([512, 480], 1, 16, 128, 64, 1),
    ([2000, 40], 1, 16, 128, 64, 1), ([1920, 60], 1, 16, 128, 128, 1)])
@torch.inference_mode()
def test_fused_is_the_three_calls(lengths, hkv, groups, dim, page, splits, neox, f32, rotary, weighed):
    """The decode layer's form against rotate_kv_write and the attention, bit for bit: outputs, cache and weights;
    one row inactive, one whose place has no page, row orders, the o_proj order."""
    b, hq = len(lengths), hkv * groups
    rotary = rotary if rotary < 64 else dim
    caches = [random_cache(lengths, hkv, dim, page, 7 + dim)[0] for _ in range(2)]
    for cache in caches:
        # a row's junk past its end is NaN; its last position is the new token's
        if b > 2:
            cache.table[2, (lengths[2] - 1) // page] = -1
    active = torch.ones(b, dtype=torch.bool, device=DEV)
    if b > 1:
        active[1] = False
    # one slice of bf16 values: the sum is the projection that rotate_kv_write is given
    heads = vectors((b, hq + 2 * hkv, dim), 3).to(DEV)
    partials = heads.float().view(1, b, -1).contiguous()
    used = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    positions = torch.randint(0, 2000, (b,), generator=gen(4)).to(DEV)
    positions[0] = 5000  # past the table: not turned
    cos_sin = rope.rotary_table(2000, rotary, 10000.0, device=DEV, dtype=torch.float32 if f32 else BF16)
    flash = PagedFlashDecode(b, hkv, groups, caches[0].capacity, DEV, num_splits=splits, head_dim=dim)
    weights = [torch.rand(b, hkv, caches[0].capacity, generator=gen(6)).to(DEV) for _ in range(2)]
    more = [dict(weights=w) if weighed else {} for w in weights]
    q, k, v = heads.split((hq, hkv, hkv), 1)
    q, _ = rope.rotate_kv_write(q, k, v, positions, active, cos_sin, caches[0], 0, at=used.long() - 1, is_neox=neox)
    exp = flash(q[:, :, None], *caches[0].layer(0), None, None, dim ** -0.5, used=used, **more[0])
    order = torch.randperm(b, generator=gen(2)).int().to(DEV)
    got = flash.fused_qkv(partials, cos_sin, positions, active, *caches[1].layer(0), dim ** -0.5, used, hq,
                          row_order=order, is_neox=neox, **more[1])
    assert torch.equal(got, exp)
    assert torch.equal(caches[1].k.view(torch.int16), caches[0].k.view(torch.int16))
    assert torch.equal(caches[1].v.view(torch.int16), caches[0].v.view(torch.int16))
    if weighed:
        assert torch.equal(*weights)
    frag = flash.fused_qkv(partials, cos_sin, positions, active, *caches[1].layer(0), dim ** -0.5, used, hq,
                           frag_out=True, is_neox=neox)
    assert torch.equal(frag.to_rows(), exp.view(b, -1))


@pytest.mark.parametrize("neox", [True, False])
@pytest.mark.parametrize("dim,rotary", [(64, 16), (64, 48), (64, 64), (128, 48), (128, 128)])
@torch.inference_mode()
def test_fused_rotation_is_the_stores(dim, rotary, neox):
    """Many pairs by an fp32 table: one rounding more or less in either kernel would show, in the cache or in rows of
    one position with V as they attend it."""
    rows, hkv, groups = 96, 5, 3
    lengths, hq = [3] * rows, 15
    caches = [random_cache(lengths, hkv, dim, 16, 7)[0] for _ in range(2)]
    heads = vectors((rows, hq + 2 * hkv, dim), 3).to(DEV)
    cos_sin = rope.rotary_table(500, rotary, 10000.0, device=DEV)
    used = torch.full((rows,), 3, dtype=torch.int32, device=DEV)
    positions = torch.randint(0, 500, (rows,), generator=gen(4)).to(DEV)
    flash = PagedFlashDecode(rows, hkv, groups, caches[0].capacity, DEV, head_dim=dim)
    q, _ = rope.rotate_kv_write(*heads.split((hq, hkv, hkv), 1), positions, None, cos_sin, caches[0], 0, at=used - 1,
                                is_neox=neox)
    exp = flash(q[:, :, None], *caches[0].layer(0), None, None, 0.3, used=used)
    got = flash.fused_qkv(heads.float().view(1, rows, -1), cos_sin, positions, None, *caches[1].layer(0), 0.3, used, hq,
                          is_neox=neox)
    assert torch.equal(caches[0].k.view(torch.int16), caches[1].k.view(torch.int16))
    assert torch.equal(got, exp)


@pytest.mark.parametrize("rows,hkv", [(70, 8), (32, 8), (33, 8), (5, 130)])
@torch.inference_mode()
def test_fused_order_of_many_rows(rows, hkv):
    """Every row once, whatever the order and however many rounds of workgroups the rows make."""
    lengths = [1 + (11 * i) % 50 for i in range(rows)]
    caches = [random_cache(lengths, hkv, 64, 16, 7)[0] for _ in range(2)]
    part = torch.randn(2, rows, 3 * hkv * 64, generator=gen(3)).to(DEV)
    cos_sin = rope.rotary_table(64, 64, 10000.0, device=DEV)
    used = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    order = torch.argsort(used, descending=True, stable=True).int()
    got = [PagedFlashDecode(rows, hkv, 1, c.capacity, DEV).fused_qkv(
        part, cos_sin, used.long() - 1, None, *c.layer(0), 0.125, used, hkv, row_order=o)
        for c, o in zip(caches, (None, order))]
    assert bool(got[0].isfinite().all()) and torch.equal(*got)
    for side in ("k", "v"):
        assert torch.equal(*(getattr(c, side).view(torch.int16) for c in caches))


@pytest.mark.parametrize("splits", [None, 3])
@torch.inference_mode()
def test_fused_row_without_a_place(splits):
    """Rows of no positions, of fewer than none and of more than the plan's or the table's: nothing is stored."""
    lengths, hkv, groups, dim = [48, 48, 96, 20, 70], 2, 3, 64
    cache, k, v, table = random_cache(lengths, hkv, dim, 16, 2)
    b, hq = len(lengths), hkv * groups
    flash = PagedFlashDecode(b, hkv, groups, cache.capacity, DEV, maximum=90, num_splits=splits)
    part = vectors((b, (hq + 2 * hkv) * dim), 1).float()[None].to(DEV)
    cos_sin = rope.rotary_table(128, 64, 10000.0, device=DEV, dtype=BF16)
    used = torch.tensor([0, -1, 91, 2 ** 31 - 1, 0], dtype=torch.int32)
    pos = used.long() - 1
    w = torch.ones(b, hkv, cache.capacity, device=DEV)
    used_dev = used.to(DEV)
    got = flash.fused_qkv(part, cos_sin, pos.to(DEV), None, *cache.layer(0), 0.125, used_dev, hq, weights=w)
    assert torch.equal(cache.k.cpu().view(torch.int16), k.view(torch.int16))
    assert torch.equal(cache.v.cpu().view(torch.int16), v.view(torch.int16))
    for i in (0, 1, 4):
        assert not got[i].any() and bool((w[i] == 1).all())
    q = part.view(b, -1, dim)[:, :hq].to(BF16)
    rope.rotary_embedding(pos.to(DEV), q, torch.zeros(b, 1, dim, dtype=BF16, device=DEV), dim, cos_sin)
    check_attention(got[2:3], q[2:3].cpu(), k[0], v[0], table[2:3], [90], 0.125)


@pytest.mark.parametrize("slices", [2, 3, 8])
@torch.inference_mode()
def test_fused_sums_slices(slices):
    """Slices in ascending order, in fp32; V rounded once."""
    b, hkv, groups, dim = 3, 2, 3, 64
    cache, k, v, table = random_cache([40, 9, 70], hkv, dim, 16, 2)
    part = torch.randn(slices, b, (hkv * groups + 2 * hkv) * dim, generator=gen(1))
    cos_sin = rope.rotary_table(128, 64, 10000.0, device=DEV)
    used = torch.tensor([40, 9, 70], dtype=torch.int32)
    flash = PagedFlashDecode(b, hkv, groups, cache.capacity, DEV)
    pos = used.long() - 1
    flash.fused_qkv(part.to(DEV), cos_sin, pos.to(DEV), None, *cache.layer(0), 0.125, used.to(DEV), hkv * groups)
    total = part[0]
    for s in range(1, slices):
        total = total + part[s]
    new_k, new_v = kv_paged.read(cache, 0, pos.to(DEV), torch.arange(b, device=DEV))
    heads = total.view(b, -1, dim)
    assert torch.equal(new_v[:, :, 0].cpu(), heads[:, -hkv:].to(BF16))
    exp = paged.rotate(heads[:, hkv * groups:-hkv], *paged.angles(pos, 64, 10000.0), True)
    got = new_k[:, :, 0].cpu().double()
    assert bool(((got - exp).abs() <= rotated_bound(heads[:, hkv * groups:-hkv], exp)).all())


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("slices", [1, 2, 5, 8])
@pytest.mark.parametrize("hkv,groups,dim,splits", [(2, 3, 64, None), (1, 16, 128, None), (2, 16, 128, 2), (2, 15, 64, 1)])
@torch.inference_mode()
def test_fused_attends_by_the_sums(hkv, groups, dim, splits, slices, f32):
    """Keys, values and results of heads summed from slices, with more channels than a workgroup's threads stage at
    once too, against rotation, store and attention of the sums. bf16 table: sums in ascending order, in fp32, rounded.
    fp32 table: multiples of 1/64 whose sums are bf16 values, so that they are what the rotation is given."""
    lengths, hq = [40, 9, 300], hkv * groups
    b = len(lengths)
    cache, k, v, table = random_cache(lengths, hkv, dim, 16, 2)
    part = torch.randn(slices, b, (hq + 2 * hkv) * dim, generator=gen(slices))
    if f32:
        part = (64 * part).round()
        part[-1] += (64 * torch.randn(part[0].shape, generator=gen(9))).round().clamp(-128, 128) - part.sum(0)
        part = part / 64
    total = part[0]
    for s in range(1, slices):
        total = total + part[s]
    heads = total.view(b, -1, dim).to(BF16)
    assert not f32 or torch.equal(heads.float(), total.view(b, -1, dim))
    cos_sin = rope.rotary_table(400, 64, 10000.0, device=DEV, dtype=torch.float32 if f32 else BF16)
    used, pos = torch.tensor(lengths, dtype=torch.int32), torch.tensor([350, 8, 299])
    flash = PagedFlashDecode(b, hkv, groups, cache.capacity, DEV, num_splits=splits, head_dim=dim)
    got = flash.fused_qkv(part.to(DEV), cos_sin, pos.to(DEV), None, *cache.layer(0), dim ** -0.5, used.to(DEV), hq)
    q, new_k, new_v = (x.clone() for x in heads.to(DEV).split((hq, hkv, hkv), 1))
    rope.rotary_embedding(pos.to(DEV), q, new_k, dim, cos_sin)
    for i, n in enumerate(lengths):
        page, place = paged.cell(table, k.shape[1], 16, i, n - 1)
        for pool, new in ((k, new_k), (v, new_v)):
            pool[0, page, :, place] = new[i].cpu()
    assert torch.equal(cache.k.cpu().view(torch.int16), k.view(torch.int16))
    assert torch.equal(cache.v.cpu().view(torch.int16), v.view(torch.int16))
    check_attention(got, q.cpu(), k[0], v[0], table, used, dim ** -0.5)


# ---------------------------------------------------------------- eviction --

@pytest.mark.parametrize("case", ["spread", "equal", "special", "negative"])
@pytest.mark.parametrize("lengths,heads,dim,page,keep,recent", [
    ([5], 1, 64, 16, 1, 0), ([40, 16, 1, 0], 2, 64, 16, 16, 4), ([33, 100], 2, 128, 32, 33, 33),
    ([1500, 1024, 1025, 700], 2, 64, 64, 1024, 100), ([4000, 2050], 1, 64, 256, 1500, 0), ([129], 3, 128, 16, 128, 1),
    ([5000, 4097, 90], 1, 64, 64, 300, 7), ([12288, 8000], 1, 64, 64, 200, 0), ([13000, 12289, 5], 2, 64, 256, 100, 1)])
@torch.inference_mode()
def test_evict(lengths, heads, dim, page, keep, recent, case):
    layers, b = 2, len(lengths)
    cache, k, v, table = random_cache(lengths, heads, dim, page, keep, layers=layers, junk=3.0)
    w = torch.randn(layers, b, heads, cache.capacity, generator=gen(keep))
    if case == "spread":
        w = torch.exp(2 * w)
    elif case == "equal":
        w = (w * 2).round() / 4
    elif case == "special":
        pick = torch.randint(0, 8, w.shape, generator=gen(1))
        for i, value in enumerate((math.nan, math.inf, -math.inf, 0.0, -0.0, -math.nan)):
            w[pick == i] = value
    keep = min(keep, cache.capacity)
    # fresh pages for what stays, in a pool that is larger by them
    need = [-(-min(n, keep) // page) for n in lengths]
    more = sum(need) + 1
    pk, pv = (torch.cat((x, torch.full((layers, more, *x.shape[2:]), 9.0, dtype=BF16)), 1).to(DEV) for x in (k, v))
    ids = (k.shape[1] + torch.randperm(more, generator=gen(2))).tolist()
    target = torch.full((b, max(1, *need)), -1, dtype=torch.int32)
    for i, n in enumerate(need):
        target[i, :n] = torch.tensor(ids[:n], dtype=torch.int32)
        ids = ids[n:]
    grown = PagedKVCache.over(pk, pv, cache.table)
    exp_k, exp_v = pk.cpu(), pv.cpu()
    used = torch.tensor(lengths, dtype=torch.int32)
    out, kept, left = kv_paged.evict(grown, w.to(DEV), used.to(DEV), keep, recent, target.to(DEV))
    assert left.tolist() == [min(n, keep) for n in lengths]
    exp_w, exp_kept = torch.zeros_like(w), torch.full((layers, b, heads, keep), -1, dtype=torch.int32)
    for layer in range(layers):
        for i, n in enumerate(lengths):
            for h in range(heads):
                stay = paged.keep(w[layer, i, h], n, keep, recent)
                exp_kept[layer, i, h, :len(stay)] = torch.tensor(stay, dtype=torch.int32)
                exp_w[layer, i, h, :len(stay)] = w[layer, i, h, stay]
                for to, j in enumerate(stay):
                    src = paged.cell(table, k.shape[1], page, i, j)
                    dst = int(target[i, to // page]), to % page
                    for side, x in ((exp_k, k), (exp_v, v)):
                        side[layer, dst[0], h, dst[1]] = x[layer, src[0], h, src[1]]
    assert torch.equal(kept.cpu(), exp_kept)
    assert torch.equal(out.cpu().view(torch.int32), exp_w.view(torch.int32))
    assert torch.equal(pk.cpu(), exp_k) and torch.equal(pv.cpu(), exp_v)
    # in place, and a target that is too short: what has no page is not copied, and nothing else is written
    w_dev = w.to(DEV)
    same, kept2, _ = kv_paged.evict(grown, w_dev, used.to(DEV), keep, recent, torch.full((b, 1), -1, dtype=torch.int32,
                                                                                           device=DEV), weights_out=w_dev)
    assert same is w_dev and torch.equal(kept2, kept)
    assert torch.equal(w_dev.cpu().view(torch.int32), exp_w.view(torch.int32))
    assert torch.equal(pk.cpu(), exp_k) and torch.equal(pv.cpu(), exp_v)


@torch.inference_mode()
def test_evict_positions_without_a_page():
    """What stays of positions without a page is zeros in the target's pages, whose former contents were others'."""
    cache, k, v, table = random_cache([80, 64], 2, 64, 16, 3, junk=3.0)
    more = torch.full((1, 12, 2, 16, 64), 9.0, dtype=BF16, device=DEV)
    pages = k.shape[1]
    line = table.clone()
    line[0, 1], line[1, 3] = -1, pages + 12
    grown = PagedKVCache.over(torch.cat((cache.k, more), 1), torch.cat((cache.v, more), 1), line.to(DEV))
    target = (pages + torch.arange(6, dtype=torch.int32)).view(2, 3)
    w = torch.rand(1, 2, 2, cache.capacity, generator=gen(4))
    before = grown.read(0)
    _, kept, left = kv_paged.evict(grown, w.to(DEV), torch.tensor([80, 64], dtype=torch.int32, device=DEV), 45, 5,
                                   target.to(DEV))
    assert left.tolist() == [45, 45]
    after = PagedKVCache.over(grown.k, grown.v, target.to(DEV)).read(0)
    for b in range(2):
        for h in range(2):
            stay = paged.keep(w[0, b, h], [80, 64][b], 45, 5)
            assert kept[0, b, h].tolist() == stay
            lost = [j for j in stay if (16 <= j < 32 if b == 0 else j >= 48)]
            assert lost
            for x, y in zip(before, after):
                assert torch.equal(x[b, h, stay], y[b, h, :45]) and not x[b, h, lost].any()
                assert bool((y[b, h, 45:48] == 9).all())


@torch.inference_mode()
def test_cache_evicts_what_has_pages():
    """``used`` past a row's pages is held to them, and a row of none stays so."""
    cache = PagedKVCache.empty(1, 3, 2, 64, 128, DEV, page=16, pages=20)
    cache.reserve([0, 1], [48, 20])
    w = torch.rand(1, 3, 2, 128, device=DEV)
    kept, left = cache.evict(w, torch.tensor([100, 100, 100], device=DEV), 40, 3)
    assert left.tolist() == [40, 32, 0] and cache.free_pages == 20 - 3 - 2 and cache.held(2) == 0
    assert kept[0, 1].tolist() == [[*range(32), *[-1] * 8]] * 2 and bool((kept[0, 2] == -1).all())


@torch.inference_mode()
def test_cache_evicts_from_long_rows_only():
    """One row over its budget and two that are not, one beginning with the other's pages, in a pool that has free
    pages for the first alone: it is held to its budget, and the others' pages, weights and contents are as they
    were."""
    cache = PagedKVCache.empty(2, 3, 2, 64, 128, DEV, page=16, pages=13)
    cache.reserve([0, 1], [100, 32])
    cache.share(2, 1, 32)
    cache.reserve(2, 40)
    assert cache.free_pages == 3
    for side, seed in ((cache.k, 3), (cache.v, 4)):
        side.copy_(vectors(side.shape, seed))
    w = torch.rand(2, 3, 2, 128, generator=gen(5))
    lengths = [97, 30, 35]
    before, table, w_dev = [cache.read(layer) for layer in range(2)], cache.table.cpu(), w.to(DEV)
    kept, left = cache.evict(w_dev, torch.tensor(lengths, dtype=torch.int32, device=DEV), 48, 4)
    assert left.tolist() == [48, 30, 35] and cache.free_pages == 7
    assert torch.equal(cache.table[1:].cpu(), table[1:])
    for layer in range(2):
        for x, y in zip(before[layer], cache.read(layer)):
            assert torch.equal(x[1:], y[1:])
            for h in range(2):
                stay = paged.keep(w[layer, 0, h], 97, 48, 4)
                assert kept[layer, 0, h].tolist() == stay and torch.equal(y[0, h, :48], x[0, h, stay])
        for row, n in enumerate(lengths):
            for h in range(2):
                stay = paged.keep(w[layer, row, h], n, 48, 4)
                exp = torch.zeros(128)
                exp[:len(stay)] = w[layer, row, h, stay]
                assert torch.equal(w_dev[layer, row, h].cpu(), exp)
                assert kept[layer, row, h].tolist() == stay + [-1] * (48 - len(stay))


@torch.inference_mode()
def test_graph_replays_of_evictions():
    """Weights and eviction recorded, with the weights read and written in place by the graph's own tensors."""
    lengths = [100, 61]
    cache, k, v, table = random_cache(lengths, 2, 64, 16, 3, capacity=112, junk=0.5)
    grown = PagedKVCache.over(*(torch.cat((x, torch.zeros_like(x)), 1) for x in (cache.k, cache.v)), cache.table)
    target = (k.shape[1] + torch.arange(4, dtype=torch.int32).view(2, 2)).to(DEV)
    used = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    w = torch.rand(1, 2, 2, 112, generator=gen(1)).to(DEV)
    kv_paged.evict(grown, w, used, 30, 4, target)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            out, kept, left = kv_paged.evict(grown, w, used, 30, 4, target)
    torch.cuda.current_stream().wait_stream(side)
    for turn in range(4):
        w.copy_(torch.rand(1, 2, 2, 112, generator=gen(turn)))
        used.sub_(7)
        for x in (grown.k, grown.v):
            x[:, k.shape[1]:] = 5
        graph.replay()
        got = [x.clone() for x in (out, kept, left, grown.k, grown.v)]
        torch.cuda.synchronize()
        for x in (grown.k, grown.v):
            x[:, k.shape[1]:] = 5
        exp = kv_paged.evict(grown, w, used, 30, 4, target)
        assert all(torch.equal(x, y) for x, y in zip(got, (*exp, grown.k, grown.v)))
        for b, n in enumerate(used.tolist()):
            for h in range(2):
                stay = paged.keep(w[0, b, h].cpu(), n, 30, 4)
                assert kept[0, b, h].tolist() == stay + [-1] * (30 - len(stay))


# ---------------------------------------------------------------- together --

@torch.inference_mode()
def test_prefill_decode_evict_decode():
    """A run of all of them: prompts are stored, steps attend and weigh, the rows are held to a budget, and steps
    go on at rotary positions past the cache's. A history in 64 bits says what each step has to give; one row
    begins with another's pages, which the eviction leaves to it."""
    hkv, groups, dim, page, steps, keep, recent = 2, 3, 64, 16, 6, 40, 8
    prompts = [70, 64, 33]
    b, hq, scale = len(prompts), hkv * groups, 0.125
    cache = PagedKVCache.empty(1, b + 1, hkv, dim, 128, DEV, page=page, pages=40)
    cache.reserve([0, 1, 2], [n + steps for n in prompts])
    cos_sin = rope.rotary_table(256, 64, 10000.0, scaling=dict(type="linear", factor=2.0), device=DEV)
    tokens = sum(prompts)
    qkv = vectors((tokens, hq + 2 * hkv, dim), 1).to(DEV)
    pos = torch.cat([torch.arange(n) for n in prompts]).to(DEV)
    slots = torch.cat([torch.full((n,), i) for i, n in enumerate(prompts)]).to(DEV)
    _, k = rope.rotate_kv_write(*qkv.split((hq, hkv, hkv), 1), pos, None, cos_sin, cache, 0, slots, keep_k=True)
    held = [[(k[slots == i][t].cpu(), qkv[slots == i][t, -hkv:].cpu()) for t in range(n)]
            for i, n in enumerate(prompts)]
    # per row and KV head: lists of (key, value), as an eviction parts them
    rows = [[[(kk[h], vv[h]) for kk, vv in held[i]] for h in range(hkv)] for i in range(b)]
    flash = PagedFlashDecode(b, hkv, groups, cache.capacity, DEV, maximum=100)
    weights = torch.zeros(1, b + 1, hkv, cache.capacity, device=DEV)
    # per row and KV head: each position's weight in 64 bits, and how far the kernel's may be off
    exact_w = [[torch.zeros(n, dtype=torch.float64) for _ in range(hkv)] for n in prompts]
    off_w = [[torch.zeros(n, dtype=torch.float64) for _ in range(hkv)] for n in prompts]
    used = torch.tensor(prompts, dtype=torch.int32, device=DEV)
    positions = used.long().clone()
    cache.share(3, 1, 64)

    def step(seed):
        nonlocal used, positions
        used = used + 1
        part = vectors((b, hq + 2 * hkv, dim), seed).float().view(1, b, -1).to(DEV)
        out = flash.fused_qkv(part, cos_sin, positions, None, *cache.layer(0), scale, used, hq, weights=weights[0])
        kv = kv_paged.read(cache, 0, used.long() - 1, cache.slots[:b])
        turned = paged.rotate(part.view(b, -1, dim).cpu()[:, :-hkv],
                              *(x / 1.0 for x in paged.angles(positions.cpu() / 2.0, 64, 10000.0)), True)
        new = turned[:, hq:]
        assert bool(((kv[0][:, :, 0].cpu().double() - new).abs()
                     <= rotated_bound(part.view(b, -1, dim).cpu()[:, hq:-hkv], new)).all())
        # the operator's own rotated bf16 query: from the rotation call
        q = part.view(b, -1, dim)[:, :hq].to(BF16)
        kk = torch.zeros(b, 1, dim, dtype=BF16, device=DEV)
        q = q.clone()
        rope.rotary_embedding(positions, q, kk, dim, cos_sin)
        for i in range(b):
            for h in range(hkv):
                rows[i][h].append((kv[0][i, h, 0].cpu(), kv[1][i, h, 0].cpu()))
                ks, vs = (torch.stack([x[s] for x in rows[i][h]]) for s in (0, 1))
                n = ks.shape[0]
                pool_k, pool_v = (torch.zeros(-(-n // 16), 1, 16, dim, dtype=BF16) for _ in range(2))
                for pool, x in ((pool_k, ks), (pool_v, vs)):
                    pool.view(-1, dim)[:n] = x
                line = torch.arange(pool_k.shape[0], dtype=torch.int32)[None]
                qi = q[i:i + 1, h * groups:(h + 1) * groups].cpu()
                p = check_attention(out[i:i + 1, h * groups:(h + 1) * groups], qi, pool_k, pool_v, line, [n], scale)[0]
                before = torch.cat((exact_w[i][h], torch.zeros(1, dtype=torch.float64)))
                tol = weight_bound(qi, pool_k, line, 0, n, scale, p, before[None] * (1 + 2.0 ** -10))[0]
                exact_w[i][h] = before + p.sum(1)[0]
                off_w[i][h] = torch.cat((off_w[i][h], torch.zeros(1, dtype=torch.float64))) + tol
                got = weights[0, i, h, :n].double().cpu()
                assert bool(((got - exact_w[i][h]).abs() <= off_w[i][h]).all())
        positions = positions + 1

    for s in range(steps):
        step(10 + s)
    lent = [x[3, :, :64].clone() for x in cache.read(0)]
    before = cache.free_pages
    kept, left = cache.evict(weights, torch.cat((used, used.new_full((1,), 64))), keep, recent, room=steps)
    assert left.tolist() == [40, 40, 39, 40] and cache.free_pages > before
    assert [cache.held(i) for i in range(4)] == [48, 48, 48, 48]
    used = left[:b].clone()
    for i in range(b):
        for h in range(hkv):
            stay = [j for j in kept[0, i, h].tolist() if j >= 0]
            assert len(stay) == int(used[i])
            assert stay[-recent:] == list(range(len(rows[i][h]) - recent, len(rows[i][h])))
            rows[i][h] = [rows[i][h][j] for j in stay]
            exact_w[i][h], off_w[i][h] = exact_w[i][h][stay], off_w[i][h][stay]
    # the row that had another's pages, and no weights of its own: the first of equals and the recent
    assert kept[0, 3].tolist() == [[*range(32), *range(56, 64)]] * hkv
    for x, y in zip(cache.read(0), lent):
        assert torch.equal(x[3, :, :40], y[:, kept[0, 3, 0].long()])
    for s in range(steps):
        step(30 + s)


@torch.inference_mode()
def test_prompt_behind_a_shared_beginning():
    """A prompt whose first pages another row holds: its other tokens are stored in pages of its own and attend the
    whole as rows of one call, the cache row's table line repeated for each."""
    hkv, groups, page, first, more = 2, 3, 16, 64, 21
    cache = PagedKVCache.empty(1, 2, hkv, 64, 128, DEV, page=page)
    cache.reserve(0, first + 5)
    cos_sin = rope.rotary_table(128, 64, 10000.0, device=DEV)
    qkv = vectors((first + 5 + more, groups * hkv + 2 * hkv, 64), 1).to(DEV)
    q, k, v = qkv.split((groups * hkv, hkv, hkv), 1)
    at = torch.arange(first + 5, device=DEV)
    rope.rotate_kv_write(q[:first + 5], k[:first + 5], v[:first + 5], at, None, cos_sin, cache, 0, torch.zeros_like(at))
    lent = [x.clone() for x in cache.read(0)]
    cache.share(1, 0, first)
    cache.reserve(1, first + more)
    at = first + torch.arange(more, device=DEV)
    turned, _ = rope.rotate_kv_write(q[-more:], k[-more:], v[-more:], at, None, cos_sin, cache, 0, torch.ones_like(at))
    assert all(torch.equal(x[0], y[0]) for x, y in zip(cache.read(0), lent))
    flash = PagedFlashDecode(more, hkv, groups, cache.capacity, DEV)
    lines = cache.table[1:].repeat(more, 1)
    got = flash(turned[:, :, None], cache.k[0], cache.v[0], lines, None, None, 0.125, used=(at + 1).int())
    check_attention(got, turned.cpu(), cache.k[0].cpu(), cache.v[0].cpu(), lines.cpu(), (at + 1).cpu(), 0.125)


@torch.inference_mode()
def test_graph_replays_follow_the_table():
    """Attention, weights and store recorded once and replayed as rows grow and their pages change, with
    eager work between the replays."""
    lengths = [30, 61]
    cache, k, v, table = random_cache(lengths, 2, 64, 16, 3, capacity=128, junk=0.5)
    q = vectors((2, 6, 64), 8)
    flash = PagedFlashDecode(2, 2, 3, cache.capacity, DEV, num_splits=3)
    eager = PagedFlashDecode(2, 2, 3, cache.capacity, DEV, num_splits=3)
    used = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    q_dev, w = q.to(DEV)[:, :, None], torch.zeros(2, 2, cache.capacity, device=DEV)
    w_out, out = torch.zeros_like(w), torch.zeros(2, 6, 1, 64, dtype=BF16, device=DEV)
    cos_sin = rope.rotary_table(256, 64, 10000.0, device=DEV)
    new = vectors((2, 10, 64), 9).to(DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    flash(q_dev, *cache.layer(0), None, None, 0.125, used=used, weights=w, weights_out=w_out)
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            turned, _ = rope.rotate_kv_write(*new.split((6, 2, 2), 1), used.long(), None, cos_sin, cache, 0,
                                             at=used.long() - 1)
            out.copy_(flash(turned[:, :, None], *cache.layer(0), None, None, 0.125, used=used, weights=w,
                            weights_out=w_out))
    torch.cuda.current_stream().wait_stream(side)
    twin = PagedKVCache.over(cache.k.clone(), cache.v.clone(), cache.table.clone())
    for turn in range(4):
        graph.replay()
        torch.cuda.synchronize()
        t, _ = rope.rotate_kv_write(*new.split((6, 2, 2), 1), used.long(), None, cos_sin, twin, 0, at=used.long() - 1)
        w2 = torch.zeros_like(w)
        exp = eager(t[:, :, None], *twin.layer(0), None, None, 0.125, used=used, weights=w, weights_out=w2)
        assert torch.equal(out, exp) and torch.equal(cache.k, twin.k)
        for i, n in enumerate(used.tolist()):
            assert torch.equal(w_out[i, :, :n], w2[i, :, :n])
        used += torch.tensor([-3, 1], dtype=torch.int32, device=DEV)
        new.mul_(1.25)
        if turn == 1:  # the pages of the rows change places
            for c in (cache, twin):
                c.table.copy_(c.table.flip(0).clone())
            used.copy_(used.flip(0).clone())


@torch.inference_mode()
def test_two_streams():
    """Two calls at once, an object each, on streams of their own."""
    cache, k, v, table = random_cache([900, 700, 800], 2, 64, 32, 3)
    used = torch.tensor([900, 700, 800], dtype=torch.int32, device=DEV)
    qs = [vectors((3, 6, 64), s).to(DEV)[:, :, None] for s in (1, 2)]
    flashes = [PagedFlashDecode(3, 2, 3, cache.capacity, DEV, num_splits=4) for _ in qs]
    alone = [f(q, *cache.layer(0), None, None, 0.125, used=used).clone() for f, q in zip(flashes, qs)]
    streams = [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    out = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                out[i].append(flashes[i](qs[i], *cache.layer(0), None, None, 0.125, used=used))
    torch.cuda.synchronize()
    assert all(torch.equal(x, alone[i]) for i in range(2) for x in out[i])


# ------------------------------------------------------------------ engine --

def small_model(seed=3, capacity=128, **over):
    cfg = preset("granite-1b", num_hidden_layers=2, vocab_size=512, **over)
    weights = synth.granite_weights(cfg, seed=seed, device=DEV)
    ep = ExpertParallel(1, 0, 4096, cfg.hidden_size, cfg.num_experts_per_tok, BF16, DEV, HipFusedExperts())
    return cfg, Granite(cfg, weights, ep, capacity)


def reserved(cfg, rows, capacity, page, positions):
    """A paged cache whose rows' pages are in no order."""
    cache = PagedKVCache(cfg, rows, capacity, DEV, BF16, page=page)
    for turn in range(0, positions, page):
        for row in reversed(range(rows)):
            cache.reserve(row, min(positions, turn + page))
    return cache


@pytest.mark.parametrize("epilogue", [True, False])
@torch.inference_mode()
def test_prefill_writes_what_the_contiguous_cache_holds(epilogue):
    """Packed and padded prefills: logits and stored positions are the contiguous cache's, bit for bit; a padded
    row's places behind its prompt are zeroed."""
    cfg, model = small_model()
    model.qkv_epilogue = epilogue
    lengths = [9, 33, 1]
    caches = [KVCache(cfg, 3, 64, DEV, BF16), reserved(cfg, 3, 64, 16, 64)]
    for c in caches:
        c.k.fill_(1)
        c.v.fill_(1)
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
            assert torch.equal(got, held)


@torch.inference_mode()
def test_prefills_keep_out_of_shared_pages():
    """A prompt into a row that begins with another's pages is refused by every prefill that goes by rows, with both
    rows as they were; into a row that has its own it is taken."""
    cfg, model = small_model()
    cache = PagedKVCache(cfg, 3, 64, DEV, BF16, page=16)
    cache.reserve([0, 2], 64)
    prompts = synth.prompts(1, [40], cfg.vocab_size, 3)
    packed_prefill_logits(model, prompts, cache)
    cache.share(1, 0, 32)
    cache.reserve(1, 64)
    before = cache.k.clone(), cache.v.clone()
    tokens = torch.tensor(prompts, device=DEV)
    columns = torch.arange(40, device=DEV)[None]
    for call in (lambda: packed_prefill_logits(model, prompts, cache, 1),
                 lambda: packed_prefill_logits(model, prompts * 2, cache, 1),
                 lambda: prefill_logits(model, prompts * 2, cache, 1),
                 lambda: model.forward(tokens, columns, columns < 40, cache, slot=0)):
        with pytest.raises(ValueError, match="shares"):
            call()
    assert torch.equal(cache.k, before[0]) and torch.equal(cache.v, before[1])
    packed_prefill_logits(model, prompts, cache, 2)
    assert all(torch.equal(x[2, :, :40], x[0, :, :40]) for layer in range(2) for x in cache.read(layer))


@torch.inference_mode()
def test_decode_layer_is_its_operators():
    """Both decode layers of the model (split-K projections with the fused attention, and the dense ones with a
    store of its own) are bit for bit the operators called one by one, an inactive row among them; and the split-K
    one's cache is the contiguous decode's."""
    cfg, model = small_model()
    b, cap, hq, hkv = 5, 64, 16, 8
    caches = [reserved(cfg, b, cap, 32, cap) for _ in range(4)]
    plain = KVCache(cfg, b, cap, DEV, BF16)
    plain.k.copy_(vectors(plain.k.shape, 1))
    plain.v.copy_(vectors(plain.v.shape, 2))
    every = torch.arange(cap, device=DEV).repeat(b), torch.arange(b, device=DEV).repeat_interleave(cap)
    for c in caches:
        for layer in range(2):
            sides = [x[layer].transpose(1, 2).reshape(b * cap, hkv, 1, 64) for x in (plain.k, plain.v)]
            c.write(layer, *sides, every[0], None, every[1])
    w = model.w["layers"][1]
    z = (vectors((b, cfg.hidden_size), 4)).to(DEV)
    positions = torch.tensor([40, 1, 0, 63, 5], device=DEV)
    active = torch.tensor([True, True, True, True, False], device=DEV)
    model.used = (positions + 1).int()
    splits = model.decode_splits(b)
    got = model.attention_splitk(z, w, caches[0], 1, positions, active, splits)
    flash = PagedFlashDecode(b, hkv, hq // hkv, cap, DEV)
    part = linear_splitk(z, w["self_attn.qkv_proj"], splits[0])
    a = flash.fused_qkv(part, model.cos_sin, positions, active, *caches[1].layer(1), cfg.attention_multiplier,
                        model.used, hq, frag_out=True)
    assert torch.equal(got, linear_splitk_frag(a, w["self_attn.o_proj"], splits[1]))
    contiguous = FlashDecode(b, hkv, hq // hkv, cap, DEV)
    contiguous.fused_qkv(part, model.cos_sin, positions, active, plain.k[1], plain.v[1], cfg.attention_multiplier,
                         model.used, hq)
    for got_side, side in zip(caches[0].read(1), (plain.k[1], plain.v[1])):
        assert torch.equal(got_side, side)
    for epilogue in (True, False):
        model.qkv_epilogue = epilogue
        got = model.attention(z, w, caches[2], 1, positions, active, positions, None)
        qkv = linear_rope_kv(z, w["self_attn.qkv_proj"], hq, hkv, positions, active, model.cos_sin, None, 1)
        heads = qkv.view(b, hq + 2 * hkv, 1, 64)
        caches[3].write(1, heads[:, hq:hq + hkv], heads[:, hq + hkv:], positions, active)
        a = flash(heads[:, :hq], *caches[3].layer(1), None, None, cfg.attention_multiplier, used=model.used)
        assert torch.equal(got, linear_dense(a.view(b, -1), w["self_attn.o_proj"]))
    for one, two in ((caches[0], caches[1]), (caches[2], caches[3])):
        assert torch.equal(one.k, two.k) and torch.equal(one.v, two.v)


@pytest.mark.parametrize("lean", [True, False])
@torch.inference_mode()
def test_decode_forward_agrees_with_the_contiguous_cache(lean):
    """A decode step through ``Granite.forward`` after a prefill: logits within the tolerance of the model's other
    paths (rel. L2 2e-2), whatever the page; a masked row's pages untouched."""
    cfg, model = small_model()
    lengths = [9, 33, 1, 40]
    caches = [KVCache(cfg, 4, 64, DEV, BF16), reserved(cfg, 4, 64, 16, 64), reserved(cfg, 4, 64, 64, 64)]
    packed, ends = build_packed(lengths, DEV)
    tokens = torch.randint(1, 512, (1, sum(lengths)), generator=gen(1)).to(DEV)
    for c in caches:
        model.forward(tokens, packed.positions[None], torch.ones_like(tokens, dtype=torch.bool), c, slot=packed,
                      last=ends.long() - 1)
    model.decode_lean = lean
    step = torch.randint(1, 512, (4, 1), generator=gen(3)).to(DEV)
    positions = torch.tensor(lengths, device=DEV)[:, None]
    valid = torch.tensor([[True], [True], [True], [False]], device=DEV)
    before = caches[1].read(1)[0][3].clone()
    logits = [model.forward(step, positions, valid, c)[:3].float() for c in caches]
    assert torch.equal(caches[1].read(1)[0][3], before)
    assert torch.equal(logits[1], logits[2])
    assert float((logits[1] - logits[0]).norm() / logits[0].norm()) < 2e-2


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("model_name", ["granite-1b", "granite-3b"])
@torch.inference_mode()
def test_engine_runs_on_the_paged_cache(page, model_name):
    """Generation over ragged prompts, a pool with pages for them and no more: the captured steps and the eager ones
    give the same tokens and the same cache, twice over, and the first tokens are the contiguous engine's."""
    cfg = preset(model_name, num_hidden_layers=2, vocab_size=512)
    weights = synth.granite_weights(cfg, seed=5, device=DEV)
    prompts = synth.prompts(5, [40, 3, 17, 64, 1], cfg.vocab_size, 7)
    runs = []
    for mode, kv_page in (("eager", page), ("graph-async", page), ("graph", page), ("eager", None)):
        ep = ExpertParallel(1, 0, 4096, cfg.hidden_size, cfg.num_experts_per_tok, BF16, DEV, HipFusedExperts())
        model = Granite(cfg, weights, ep, 128)
        requests = [Request(str(i), p, 12) for i, p in enumerate(prompts)]
        run = OptimizedEngine(model, requests, mode=mode, ignore_eos=True, kv_page=kv_page, capacity=128)
        first, _ = run.generate()
        second, _ = run.generate()
        assert first == second and all(len(o) == 12 for o in first.values())
        assert kv_page is None or run.cache.free_pages == 0
        runs.append((first, run.cache.k.clone(), run.cache.v.clone()))
    for other in runs[1:3]:
        assert other[0] == runs[0][0]
        assert torch.equal(other[1], runs[0][1]) and torch.equal(other[2], runs[0][2])
    assert all(runs[3][0][r][0] == o[0] for r, o in runs[0][0].items())


@pytest.mark.parametrize("kind", [Engine, BatchPrefillEngine])
@torch.inference_mode()
def test_every_engine_takes_the_paged_cache(kind):
    """The engines without the optimized policy: eager and captured steps agree, and the first tokens are the
    contiguous cache's; a capacity that is no multiple of the page."""
    cfg, _ = small_model()
    prompts = synth.prompts(3, [5, 21, 9], cfg.vocab_size, 7)
    runs = []
    for mode, kv_page in (("eager", 16), ("graph", 16), ("eager", None)):
        model = small_model()[1]
        run = kind(model, [Request(str(i), p, 6) for i, p in enumerate(prompts)], mode=mode, ignore_eos=True,
                   kv_page=kv_page, capacity=40)
        out, _ = run.generate()
        assert all(len(o) == 6 for o in out.values())
        runs.append((out, run.cache.k.clone()))
    assert runs[0][0] == runs[1][0] and torch.equal(runs[0][1], runs[1][1])
    assert all(runs[2][0][r][0] == o[0] for r, o in runs[0][0].items())


@torch.inference_mode()
def test_decode_attention_of_the_other_cache_is_refused():
    cfg, model = small_model()
    token, valid = torch.ones(2, 1, dtype=torch.int64, device=DEV), torch.ones(2, 1, dtype=torch.bool, device=DEV)
    caches = [KVCache(cfg, 2, 64, DEV, BF16), QuantKVCache(cfg, 2, 64, DEV, BF16), reserved(cfg, 2, 64, 16, 8)]
    flashes = [FlashDecode(2, 8, 2, 64, DEV), QuantFlashDecode(2, 8, 2, 64, DEV), PagedFlashDecode(2, 8, 2, 64, DEV)]
    for i, flash in enumerate(flashes):
        model.decode_flash = flash
        for j, cache in enumerate(caches):
            if i != j:
                with pytest.raises(ValueError, match="another KV cache type"):
                    model.forward(token, token - 1, valid, cache)
        model.forward(token, token - 1, valid, caches[i])


# ---------------------------------------------------------------- refusals --

@torch.inference_mode()
def test_refusals():
    cache, *_ = random_cache([20, 9], 2, 64, 16, 1)
    flash = PagedFlashDecode(2, 2, 3, cache.capacity, DEV)
    layer = cache.layer(0)
    q = torch.zeros(2, 6, 1, 64, dtype=BF16, device=DEV)
    used = torch.tensor([20, 9], dtype=torch.int32, device=DEV)
    w = torch.zeros(2, 2, cache.capacity, device=DEV)
    good = dict(used=used)
    for args, more, text in [
            ((q.half(), *layer), good, "BF16"), ((q[:, :4], *layer), good, "heads"),
            ((q[..., :32], *layer), good, "head_dim"), ((q.cpu(), *layer), good, "one device"),
            ((q, layer.k.float(), layer.v, layer.table), good, "BF16"),
            ((q, layer.k, layer.v, layer.table.long()), good, "int32"),
            ((q, layer.k, layer.v, layer.table[:1]), good, "another batch"),
            ((q, layer.k, layer.v, layer.table[:, :1].contiguous()), good, "another batch"),
            ((q, layer.k, layer.v, layer.table.cpu()), good, "ROCm device"),
            ((q, *layer), dict(used=used[:1]), "one entry per row"),
            ((q, *layer), dict(used=used, weights=w.half()), "fp32"),
            ((q, *layer), dict(used=used, weights=w[..., 1:]), "fp32"),
            ((q, *layer), dict(used=used, weights_out=w), "goes with")]:
        with pytest.raises(ValueError, match=text):
            flash(*args, None, None, 0.125, **more)
    part = torch.zeros(1, 2, 10 * 64, device=DEV)
    cos_sin, pos = rope.rotary_table(64, 64, 10000.0, device=DEV), used.long()
    for p, t, text in [(part.half(), cos_sin, "fp32"), (part[..., 1:], cos_sin, "partials"),
                       (part, cos_sin.double(), "FP32 or BF16"), (part, cos_sin.cpu(), "device"),
                       (part, cos_sin[:, :40].contiguous(), "multiple of 16"), (part, cos_sin[:, 1:], "contiguous")]:
        with pytest.raises(ValueError, match=text):
            flash.fused_qkv(p, t, pos, None, *layer, 0.125, used, 6)
    x = torch.zeros(2, 2, 1, 64, dtype=BF16, device=DEV)
    for k, text in [(x.float(), "BF16"), (x[:, :1], "heads"), (x.cpu(), "device"), (x[:, :, :, :32], "heads")]:
        with pytest.raises(ValueError, match=text):
            cache.write(0, k, k, pos, None)
    with pytest.raises(ValueError, match="keeps"):
        kv_paged.evict(cache, torch.zeros(1, 2, 2, cache.capacity, device=DEV), used, 4, 5, layer.table)
    with pytest.raises(ValueError, match="Weights"):
        kv_paged.evict(cache, torch.zeros(1, 2, 2, 5, device=DEV), used, 4, 2, layer.table)
    with pytest.raises(ValueError, match="line per row"):
        kv_paged.evict(cache, torch.zeros(1, 2, 2, cache.capacity, device=DEV), used, 4, 2, layer.table[:1])
    both = torch.zeros(9, 2, 2, cache.capacity, device=DEV)
    with pytest.raises(NativeError):
        flash(q, *layer, None, None, 0.125, used=used, weights=both[0], weights_out=both.view(-1, 2, cache.capacity)[1:3])
    two = PagedKVCache.empty(2, 2, 2, 64, cache.capacity, DEV, page=16)
    with pytest.raises(NativeError):
        kv_paged.evict(two, both[:2], used, 4, 2, layer.table, weights_out=both[1:3])
    turned = x[:, :, 0]
    for t in (turned[:1].expand(2, -1, -1), turned[..., 1:33], turned[:, :, ::2]):
        with pytest.raises(ValueError, match="in place"):
            rope.rotary_embedding(pos, t, turned.clone(), t.shape[-1], rope.rotary_table(64, 32, 10000.0, device=DEV))
    # the buffers of the refused calls are as they were
    assert not both.any() and not turned.any()
    assert bool((w == 0).all())
