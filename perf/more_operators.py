"""The paged KV cache: its store with rotary positions, the decode attention that reads it, and eviction.

Keys and values ``[layers, pages, kv_heads, page, D]`` lie in pages of a pool; a table ``[rows, width]`` names the
pages of each row (-1: none). Five passes:

* ``store``: queries and keys of new tokens are rotated (pairs in halves or interleaved, all of the head's channels
  or the first ``rotary``, positions as they are or scaled for long contexts), keys and values go to their pages
  (``rope.rotate_kv_write``);
* ``attn``: one query token per row attends the first ``used[b]`` positions of its row
  (``flash_decode.PagedFlashDecode``), ``used`` 0 giving zeros;
* ``fused``: the decode layer's form. The packed QKV projection arrives as fp32 partials; they are summed, rotated
  and rounded to bf16, the new token's key and value go to position ``used[b] - 1``, and the query attends the row
  with them (``PagedFlashDecode.fused_qkv``). Rotation goes by a position of its own, which after an eviction is
  past the place in the cache;
* ``weigh``: ``attn``, and each position's probability, summed over the query heads of its KV head, is added to a
  running weight;
* ``evict``: of each row, layer and KV head the ``recent`` newest positions and the heaviest of the others stay,
  ``keep`` in all, and go in their order to fresh pages with their weights (``kv_paged.evict``).

Heads, rows and contexts are those of the two configuration presets (24 or 16 query heads over 8 KV heads of 64
channels) and of the attention tests, one user to 128 rows, contexts to 4096, and generic long contexts and heads
of 128 channels. Decode cases run several layers, each with a cache of its own, as a model's step does.
"""
import math

import numpy as np
import torch

own = False

DEVICE = "cuda:0"
BF16 = torch.bfloat16
THETA = 10000.0
TRAINED = 4096          # positions that the unscaled frequencies were made for
FACTOR = 8.0            # how much further a scaled table reaches


def listed():
    return [
        # The store of one decode step of the headline batch: 64 tokens, one per row; latency counts.
        dict(name="store_b64", op="store", dim=64, rotary=64, neox=True, scaling="none", kv_heads=8, groups=3, page=64,
             rows=64, low=1, high=1),
        # One ordinary prompt of 700 tokens of the small model; interleaved pairs, half of the head rotated.
        dict(name="store_prompt_700", op="store", dim=64, rotary=32, neox=False, scaling="linear", kv_heads=8,
             groups=2, page=16, rows=1, low=700, high=700),
        # A packed prefill of 48 ragged prompts (about 50,000 tokens), frequencies scaled for long contexts.
        dict(name="store_prefill_48_ragged", op="store", dim=64, rotary=64, neox=True, scaling="yarn", kv_heads=8,
             groups=3, page=64, rows=48, low=64, high=2048),
        # One user of the small model in a short chat, small pages.
        dict(name="attn_b1_509", op="attn", dim=64, kv_heads=8, groups=2, page=16, layers=4, rows=1, low=509,
             high=509),
        # Long-context serving: the largest batch over ragged contexts, bound by the KV stream.
        dict(name="attn_b128_ragged", op="attn", dim=64, kv_heads=8, groups=3, page=64, layers=2, rows=128, low=1024,
             high=4095),
        # A few documents of up to 32768 tokens, heads of 128 channels: the key range has to be split.
        dict(name="attn_b8_32768", op="attn", dim=128, kv_heads=8, groups=4, page=256, layers=1, rows=8, low=8191,
             high=32768),
        # The decode layer of one user: reduction, rotation, store and attention.
        dict(name="fused_b1_1000", op="fused", dim=64, rotary=64, neox=True, scaling="none", kv_heads=8, groups=3,
             page=16, layers=4, rows=1, low=1000, high=1000),
        # The headline decode layer: 64 rows in their second thousand of tokens.
        dict(name="fused_b64", op="fused", dim=64, rotary=64, neox=True, scaling="yarn", kv_heads=8, groups=3, page=64,
             layers=4, rows=64, low=1025, high=1279),
        # A few users whose long rows are weighed for an eviction.
        dict(name="weigh_b3_long", op="weigh", dim=64, kv_heads=8, groups=2, page=32, layers=4, rows=3, low=2049,
             high=4001),
        # The headline batch, weighed.
        dict(name="weigh_b64", op="weigh", dim=64, kv_heads=8, groups=3, page=64, layers=4, rows=64, low=1025,
             high=1279),
        # Four chats of the small model go back to 512 positions.
        dict(name="evict_b4_to_512", op="evict", dim=64, kv_heads=8, page=16, layers=4, rows=4, low=600, high=700,
             keep=512, recent=64),
        # Sixteen long rows go back to 1024 positions, in eight layers.
        dict(name="evict_b16_to_1024", op="evict", dim=64, kv_heads=8, page=64, layers=8, rows=16, low=2049,
             high=4095, keep=1024, recent=128),
    ]


def _log_int(rng, low, high):
    return min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1))) - 0.5)) or low)


def draw(rng):
    op = rng.choice(["store", "attn", "attn", "fused", "weigh", "evict"])
    case = dict(op=op, dim=rng.choice([64, 64, 128]), kv_heads=rng.choice([1, 2, 8, 8]),
                page=rng.choice([16, 32, 64, 128, 256]))
    if op in ("store", "fused"):
        case.update(rotary=rng.choice([case["dim"], case["dim"], 32, 48]), neox=rng.random() < 0.6,
                    scaling=rng.choice(["none", "linear", "yarn"]))
    if op != "evict":
        case["groups"] = rng.choice([1, 2, 2, 3, 3, 4, 6, 8, 16])
    wide = case["kv_heads"] * case["dim"] // 64
    if op == "store":
        rows = _log_int(rng, 1, 128)
        high = _log_int(rng, 1, max(1, min(4095, 400000 // (rows * wide * (case["groups"] + 2)))))
        case.update(rows=rows, low=max(1, int(high * rng.uniform(0.1, 1.0))), high=high)
        return case
    rows = _log_int(rng, 1, 128)
    if op == "evict":
        rows = min(rows, 32)
        high = _log_int(rng, 2, max(2, min(8191, 262144 // (rows * wide))))
        keep = _log_int(rng, 1, high)
        case.update(layers=rng.randint(1, 4), rows=rows, low=max(1, int(high * rng.uniform(0.3, 1.0))), high=high,
                    keep=keep, recent=int(keep * rng.choice([0.0, 0.1, 0.5, 1.0])))
        return case
    high = _log_int(rng, 1, max(1, min(32768, 2400000 // (rows * wide))))
    low = int(high * rng.uniform(0.1, 1.0))
    if op == "fused":
        low = max(1, low)           # the new token is attended, so a row holds one at least
    elif rng.random() < 0.3:
        low = 0                     # rows that hold nothing yet
    case.update(layers=1 if rows * high * wide > 400000 else rng.randint(1, 4), rows=rows, low=low, high=high)
    return case


# ---------------------------------------------------------------- inputs --

def _lengths(case):
    return np.rint(np.linspace(case["low"], case["high"], case["rows"])).astype(np.int64)


class _Inputs:
    """Tensors from one seed, on the GPU."""

    def __init__(self, seed):
        self.gen = torch.Generator(device=DEVICE)
        self.gen.manual_seed(seed)
        self.rng = np.random.RandomState(seed % (1 << 32))

    def normal(self, *shape, std=1.0):
        return torch.empty(*shape, device=DEVICE, dtype=torch.float32).normal_(0.0, std, generator=self.gen)

    def vectors(self, *shape):
        """Keys or values: channels of unequal size, as a model's have, a few of them several times the others."""
        spread = torch.exp(self.normal(shape[-1], std=0.5))
        return (self.normal(*shape) * spread).to(BF16)

    def lengths(self, case):
        return self.rng.permutation(_lengths(case))

    def tables(self, page, width, *counts):
        """For each of ``counts`` (positions per row) a table ``[rows, width]``; all of them share one pool, its
        pages in no order. Returns the tables and the pool's number of pages."""
        need = [-(-c // page) for c in counts]
        total = int(sum(n.sum() for n in need)) + 2
        ids, at, out = self.rng.permutation(total).astype(np.int32), 0, []
        for n in need:
            t = np.full((len(n), width), -1, np.int32)
            seen = np.arange(width)[None] < n[:, None]
            t[seen] = ids[at:at + int(n.sum())]
            at += int(n.sum())
            out.append(torch.from_numpy(t).to(DEVICE))
        return out, total


def _frequencies(rotary, scaling):
    """Radians a position moves each pair, in 64 bits, and the factor of the rotated values."""
    i = torch.arange(rotary // 2, device=DEVICE, dtype=torch.float64)
    inv = THETA ** (-2 * i / rotary)
    if scaling == "none":
        return inv, 1.0
    if scaling == "linear":
        return inv / FACTOR, 1.0
    # YaRN: pairs that turn often within the trained positions keep their frequency, those that turn less than
    # once are interpolated, and between the two lies a ramp over the pair's index
    def index(turns):
        return rotary * math.log(TRAINED / (turns * 2 * math.pi)) / (2 * math.log(THETA))
    low, high = max(math.floor(index(32.0)), 0), min(math.ceil(index(1.0)), rotary - 1)
    ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
    return inv * (1 - ramp) + inv / FACTOR * ramp, 0.1 * math.log(FACTOR) + 1


def _table(case, length):
    """cos | sin ``[length, rotary]``, formed in 64 bits and held in 32."""
    inv, factor = _frequencies(case["rotary"], case["scaling"])
    angle = torch.arange(length, device=DEVICE, dtype=torch.float64)[:, None] * inv
    return (torch.cat((angle.cos(), angle.sin()), -1) * factor).float()


def _pool(inp, layers, pages, case):
    """Random keys or values of every page, one layer after the other."""
    shape = (pages, case["kv_heads"], case["page"], case["dim"])
    out = torch.empty(layers, *shape, device=DEVICE, dtype=BF16)
    for layer in range(layers):
        for at in range(0, pages, 4096):
            out[layer, at:at + 4096] = inp.vectors(min(4096, pages - at), *shape[1:])
    return out


def prepare(case, seed):
    inp = _Inputs(seed)
    lengths, page, dim, hkv = inp.lengths(case), case["page"], case["dim"], case["kv_heads"]
    rows = case["rows"]
    if case["op"] == "store":
        # packed tokens as a prefill's QKV projection leaves them: q, k and v heads are columns of one row
        tokens, hq = int(lengths.sum()), hkv * case["groups"]
        decode = case["high"] == 1
        held = np.full(rows, 1280) if decode else lengths
        (table,), pages = inp.tables(page, -(-int(held.max()) // page), held)
        qkv = inp.vectors(tokens, hq + 2 * hkv, dim)
        positions = (inp.rng.randint(0, 1280, tokens) if decode    # a decode step's tokens lie anywhere in their rows
                     else np.concatenate([np.arange(n) for n in lengths]))
        q, k, v = qkv.split((hq, hkv, hkv), 1)
        pool = torch.zeros(2, 1, pages, hkv, page, dim, device=DEVICE, dtype=BF16)
        return dict(case=case, q=q, k=k, v=v, positions=torch.from_numpy(positions).to(DEVICE),
                    slots=torch.from_numpy(np.repeat(np.arange(rows), lengths)).to(DEVICE), pk=pool[0], pv=pool[1],
                    table=table, cos_sin=_table(case, int(positions.max()) + 1))
    if case["op"] == "evict":
        width = -(-int(lengths.max()) // page)
        (table, target), pages = inp.tables(page, width, lengths, np.minimum(lengths, case["keep"]))
        # accumulated weights: a few positions hold most of it
        weights = torch.exp(inp.normal(case["layers"], rows, hkv, width * page, std=2.0))
        return dict(case=case, pk=_pool(inp, case["layers"], pages, case), pv=_pool(inp, case["layers"], pages, case),
                    table=table, target=target, used=torch.from_numpy(lengths).to(DEVICE, torch.int32), weights=weights)
    width = max(1, -(-int(lengths.max()) // page))
    (table,), pages = inp.tables(page, width, lengths)
    used = torch.from_numpy(lengths).to(DEVICE, torch.int32)
    s = dict(case=case, pk=_pool(inp, case["layers"], pages, case), pv=_pool(inp, case["layers"], pages, case),
             table=table, used=used, scale=1.0 / math.sqrt(dim))
    hq = hkv * case["groups"]
    if case["op"] != "fused":
        s["q"] = [(1.5 * inp.normal(rows, hq, 1, dim)).to(BF16) for _ in range(case["layers"])]
        if case["op"] == "weigh":
            shape = (case["layers"], rows, hkv, width * page)
            # what a few earlier steps left
            s["before"], s["after"] = 0.01 * torch.exp(inp.normal(*shape)), torch.zeros(*shape, device=DEVICE)
        return s
    # three K slices of the packed projection; query columns larger, so that scores spread as a trained model's do
    size = torch.ones((hq + 2 * hkv) * dim, device=DEVICE)
    size[:hq * dim] = 1.5
    s["partials"] = [inp.normal(3, rows, size.numel(), std=3 ** -0.5) * size for _ in range(case["layers"])]
    s["positions"] = used.long() - 1 + torch.from_numpy(inp.rng.randint(0, 1024, rows)).to(DEVICE)
    s["cos_sin"] = _table(case, int(s["positions"].max()) + 1)
    # a ragged batch's rows are dispatched longest first, as the engine has it
    ragged = case["high"] > 1.25 * case["low"]
    s["order"] = torch.argsort(used, descending=True, stable=True).int() if ragged else None
    return s


# ------------------------------------------------------- the framework's --

def _own_cache(s):
    from litemoe_amd.cache import PagedKVCache
    if "cache" not in s:
        s["cache"] = PagedKVCache.over(s["pk"], s["pv"], s["table"])
    return s["cache"]


def _own_flash(s):
    from litemoe_amd.flash_decode import PagedFlashDecode
    if "flash" not in s:
        case = s["case"]
        capacity = s["table"].shape[1] * case["page"]
        s["flash"] = PagedFlashDecode(case["rows"], case["kv_heads"], case["groups"], capacity, DEVICE,
                                      min(capacity, max(1, case["high"])), head_dim=case["dim"])
    return s["flash"]


def _own_run(s):
    from litemoe_amd import kv_paged, rope
    case, cache = s["case"], _own_cache(s)
    if case["op"] == "store":
        q, k = rope.rotate_kv_write(s["q"], s["k"], s["v"], s["positions"], None, s["cos_sin"], cache, 0, s["slots"],
                                    is_neox=case["neox"], keep_k=case["high"] > 1)
        return [q, s["pk"], s["pv"]] + ([k] if case["high"] > 1 else [])
    if case["op"] == "evict":
        weights, kept, used = kv_paged.evict(cache, s["weights"], s["used"], case["keep"], case["recent"], s["target"])
        return weights, kept, used, s["pk"], s["pv"]
    flash, out = _own_flash(s), []
    for layer in range(case["layers"]):
        held = cache.layer(layer)
        if case["op"] == "attn":
            out.append(flash(s["q"][layer], *held, None, None, s["scale"], used=s["used"]))
        elif case["op"] == "weigh":
            a = flash(s["q"][layer], *held, None, None, s["scale"], used=s["used"], weights=s["before"][layer],
                      weights_out=s["after"][layer])
            out.append((a, s["after"][layer]))
        else:
            a = flash.fused_qkv(s["partials"][layer], s["cos_sin"], s["positions"], None, *held, s["scale"], s["used"],
                                case["kv_heads"] * case["groups"], row_order=s["order"], is_neox=case["neox"])
            out.append((a, *kv_paged.read(cache, layer, s["used"] - 1, cache.slots)))
    return out


# ----------------------------------------------------------- plain forms --

def _rotate(x, cos_sin, neox):
    """``x [T, heads, D]`` with its first ``R`` channels rotated by ``cos_sin [T, R]``, in fp32."""
    r = cos_sin.shape[-1]
    cos, sin = cos_sin[:, None].chunk(2, -1)
    turned, rest = x[..., :r].float(), x[..., r:].float()
    x1, x2 = turned.chunk(2, -1) if neox else (turned[..., 0::2], turned[..., 1::2])
    o = (x1 * cos - x2 * sin, x2 * cos + x1 * sin)
    o = torch.cat(o, -1) if neox else torch.stack(o, -1).flatten(-2)
    return torch.cat((o, rest), -1)


def _place(table, rows, at, page):
    """Page and place in it of positions ``at`` of ``rows``."""
    return table[rows, at // page].long(), at % page


def _rows_of(pool, table):
    """Each row's positions, one after the other: ``[B, H, C, D]`` in fp32."""
    x = pool[table.clamp(min=0).long()]
    return x.permute(0, 2, 1, 3, 4).flatten(2, 3).float()


def _attend(q, k, v, used, scale):
    """``q [B, H, G, D]`` over ``k, v [B, H, C, D]`` in fp32: the result and the probabilities; a row with nothing
    used gives zeros."""
    seen = torch.arange(k.shape[2], device=DEVICE)[None] < used[:, None]
    scores = (torch.matmul(q, k.transpose(-1, -2)) * scale).masked_fill(~seen[:, None, None], -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True).clamp(min=-1e30))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-30)
    return torch.matmul(p, v), p


def _plain_evict(s):
    case, page = s["case"], s["case"]["page"]
    keep, recent, used = case["keep"], case["recent"], s["used"]
    layers, rows, heads, capacity = s["weights"].shape
    slot = torch.arange(capacity, device=DEVICE)[None]
    live, newest = slot < used[:, None], slot >= used[:, None] - recent
    rank = s["weights"].masked_fill((live & newest)[:, None], math.inf).masked_fill(~live[:, None], -math.inf)
    kept = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :keep]
    left = used.clamp(max=keep)
    there = torch.arange(keep, device=DEVICE)[None] < left[:, None]
    kept = kept.masked_fill(~there[:, None], capacity).sort(-1).values
    kept = kept.masked_fill(~there[:, None], -1)
    weights = torch.zeros_like(s["weights"])
    weights[..., :keep] = torch.gather(s["weights"], -1, kept.clamp(min=0)) * there[:, None]
    row, to = there.nonzero(as_tuple=True)                     # every kept place of every row
    new_page, new_place = _place(s["target"], row, to, page)
    at = kept[:, row, :, to]                                   # [places, L, H]
    old_page, old_place = _place(s["table"], row[:, None, None], at, page)
    layer, head = torch.arange(layers, device=DEVICE)[:, None], torch.arange(heads, device=DEVICE)
    for pool in (s["pk"], s["pv"]):
        pool[layer, new_page[:, None, None], head, new_place[:, None, None]] = pool[layer, old_page, head, old_place]
    return weights, kept.int(), left, s["pk"], s["pv"]


def _plain_run(s):
    case, page, dim = s["case"], s["case"]["page"], s["case"]["dim"]
    if case["op"] == "evict":
        return _plain_evict(s)
    rows, hkv, groups = case["rows"], case["kv_heads"], case.get("groups")
    if case["op"] == "store":
        cos_sin = s["cos_sin"][s["positions"]]
        q, k = (_rotate(x, cos_sin, case["neox"]).to(BF16) for x in (s["q"], s["k"]))
        at, place = _place(s["table"], s["slots"], s["positions"], page)
        s["pk"][0, at, :, place] = k
        s["pv"][0, at, :, place] = s["v"]
        return [q, s["pk"], s["pv"]] + ([k] if case["high"] > 1 else [])
    out = []
    for layer in range(case["layers"]):
        pk, pv = s["pk"][layer], s["pv"][layer]
        if case["op"] != "fused":
            q = s["q"][layer]
        else:
            p = s["partials"][layer]
            qkv = ((p[0] + p[1]) + p[2]).view(rows, -1, dim)
            cos_sin = s["cos_sin"][s["positions"]]
            q = _rotate(qkv[:, :hkv * groups], cos_sin, case["neox"]).to(BF16)
            k, v = _rotate(qkv[:, hkv * groups:-hkv], cos_sin, case["neox"]).to(BF16), qkv[:, -hkv:].to(BF16)
            at, place = _place(s["table"], torch.arange(rows, device=DEVICE), s["used"].long() - 1, page)
            pk[at, :, place], pv[at, :, place] = k, v
        a, p = _attend(q.view(rows, hkv, groups, dim).float(), _rows_of(pk, s["table"]), _rows_of(pv, s["table"]),
                       s["used"], s["scale"])
        a = a.to(BF16).view(rows, hkv * groups, 1, dim)
        if case["op"] == "weigh":
            seen = torch.arange(p.shape[-1], device=DEVICE)[None] < s["used"][:, None]
            s["after"][layer].copy_(torch.where(seen[:, None], s["before"][layer] + p.sum(2), s["after"][layer]))
            a = (a, s["after"][layer])
        elif case["op"] == "fused":
            a = (a, pk[at, :, place][:, :, None], pv[at, :, place][:, :, None])
        out.append(a)
    return out


def run(state):
    return _own_run(state) if own else _plain_run(state)


# ------------------------------------------------------- work and 64 bits --

def work(case):
    dim, hkv, rows = case["dim"], case["kv_heads"], case["rows"]
    lengths = _lengths(case)
    total, token = int(lengths.sum()), hkv * dim * 4         # K and V of one position
    if case["op"] == "evict":
        kept = int(np.minimum(lengths, case["keep"]).sum())
        # the weights in, the kept positions in and out, their weights and indices out, the tables
        size = hkv * (total * 4 + kept * 8) + kept * token * 2
        return dict(bytes=case["layers"] * size + (total + kept) // case["page"] * 4, flops=case["layers"] * hkv * total)
    hq = hkv * case["groups"]
    if case["op"] == "store":
        # q, k and v in and out (a prompt's k also for its own attention), the angles, a position and a slot
        heads = 2 * (hq + 2 * hkv) + (hkv if case["high"] > 1 else 0)
        return dict(bytes=total * (heads * dim * 2 + case["rotary"] * 4 + 16), flops=total * (hq + hkv) * dim * 3)
    size, flops = total * (token + 4 / case["page"]) + rows * 4, total * hq * dim * 4
    if case["op"] == "fused":
        size += rows * ((hq + 2 * hkv) * dim * 12 + hq * dim * 2 + case["rotary"] * 4 + 8 + 2 * token)
        flops += rows * (hq + 2 * hkv) * dim * 8
    else:
        size += rows * hq * dim * 4
    if case["op"] == "weigh":
        size += total * hkv * 8
        flops += total * hq
    return dict(bytes=case["layers"] * size, flops=case["layers"] * flops)


def _angles64(case, positions):
    """``cos, sin [T, rotary / 2]`` in 64 bits from the definition."""
    r, out = case["rotary"], []
    for i in range(r // 2):
        f = THETA ** (-2.0 * i / r)
        if case["scaling"] == "linear":
            f = f / FACTOR
        elif case["scaling"] == "yarn":
            # turns of the pair's index within the trained positions decide where the ramp lies
            first = max(math.floor(r * math.log(TRAINED / (64 * math.pi)) / (2 * math.log(THETA))), 0)
            last = min(math.ceil(r * math.log(TRAINED / (2 * math.pi)) / (2 * math.log(THETA))), r - 1)
            share = min(1.0, max(0.0, (i - first) / max(last - first, 0.001)))
            f = f * (1 - share) + f / FACTOR * share
        out.append(positions.double() * f)
    size = 1 + 0.1 * math.log(FACTOR) if case["scaling"] == "yarn" else 1.0
    angle = torch.stack(out, -1)
    return size * torch.cos(angle), size * torch.sin(angle)


def _rotated64(x, cos, sin, neox):
    o, r = x.double().clone(), 2 * cos.shape[-1]
    a, b = (slice(0, r // 2), slice(r // 2, r)) if neox else (slice(0, r, 2), slice(1, r, 2))
    x1, x2 = o[..., a].clone(), o[..., b].clone()
    o[..., a] = x1 * cos[:, None] - x2 * sin[:, None]
    o[..., b] = x1 * sin[:, None] + x2 * cos[:, None]
    return o


def _row64(pool, table, row, n, page):
    """The first ``n`` positions of a row: ``[H, n, D]`` in 64 bits."""
    pages = [int(p) for p in table[row, :-(-n // page)].tolist()]
    return torch.cat([pool[p].double() for p in pages], 1)[:, :n]


def _exact_evict(s):
    case, page = s["case"], s["case"]["page"]
    used, table, target = s["used"].tolist(), s["table"].tolist(), s["target"].tolist()
    host = s["weights"].cpu().numpy()
    layers, rows, heads, _ = host.shape
    weights = np.zeros(host.shape)
    kept = np.full((layers, rows, heads, case["keep"]), -1, np.int32)
    pools = [s["pk"].double(), s["pv"].double()]
    for b, n in enumerate(used):
        new = [target[b][i // page] * page + i % page for i in range(min(n, case["keep"]))]
        old = np.asarray([table[b][i // page] * page + i % page for i in range(n)])
        for layer in range(layers):
            for h in range(heads):
                w = host[layer, b, h, :n]
                free = max(n - case["recent"], 0) if n > case["keep"] else 0
                heavy = np.argsort(-w[:free].astype(np.float64), kind="stable")[:len(new) - (n - free)]
                chosen = np.sort(np.concatenate((heavy, np.arange(free, n)))).astype(np.int64)
                kept[layer, b, h, :len(chosen)] = chosen
                weights[layer, b, h, :len(chosen)] = w[chosen]
                for pool, source in zip(pools, (s["pk"], s["pv"])):
                    src = torch.from_numpy(old[chosen]).to(DEVICE)
                    dst = torch.tensor(new, device=DEVICE, dtype=torch.int64)
                    pool[layer, dst // page, h, dst % page] = source[layer, src // page, h, src % page].double()
    return (torch.from_numpy(weights), torch.from_numpy(kept),
            torch.tensor([min(n, case["keep"]) for n in used], dtype=torch.int32), *pools)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "evict":
        return _exact_evict(s)
    rows, hkv, dim, page = case["rows"], case["kv_heads"], case["dim"], case["page"]
    groups = case["groups"]
    if case["op"] == "store":
        cos, sin = _angles64(case, s["positions"])
        q, k = (_rotated64(s[x], cos, sin, case["neox"]) for x in ("q", "k"))
        pk, pv = s["pk"].double(), s["pv"].double()
        pages = s["table"].long()[s["slots"], s["positions"] // page]
        for h in range(hkv):
            pk[0, pages, h, s["positions"] % page] = k[:, h]
            pv[0, pages, h, s["positions"] % page] = s["v"][:, h].double()
        return [q, pk, pv] + ([k] if case["high"] > 1 else [])
    out = []
    for layer in range(case["layers"]):
        a = torch.zeros(rows, hkv * groups, 1, dim, dtype=torch.float64, device=DEVICE)
        new_k, new_v = (torch.zeros(rows, hkv, 1, dim, dtype=torch.float64, device=DEVICE) for _ in range(2))
        if case["op"] == "weigh":
            after = torch.zeros(rows, hkv, s["table"].shape[1] * page, dtype=torch.float64, device=DEVICE)
        for b, n in enumerate(s["used"].tolist()):
            if not n:
                continue
            k, v = (_row64(s[x][layer], s["table"], b, n, page) for x in ("pk", "pv"))
            if case["op"] != "fused":
                q = s["q"][layer][b].double().view(hkv, groups, dim)
            else:
                heads = s["partials"][layer][:, b].double().sum(0).view(1, -1, dim)
                cos, sin = _angles64(case, s["positions"][b:b + 1])
                # the rotated query and the new token's key and value are the operator's own bf16
                turned = _rotated64(heads[:, :-hkv], cos, sin, case["neox"])[0]
                new_k[b, :, 0], new_v[b, :, 0] = turned[hkv * groups:], heads[0, -hkv:]
                q = turned[:hkv * groups].to(BF16).double().view(hkv, groups, dim)
                k[:, n - 1], v[:, n - 1] = new_k[b, :, 0].to(BF16).double(), new_v[b, :, 0].to(BF16).double()
            p = torch.softmax(q @ k.transpose(1, 2) * s["scale"], -1)
            a[b, :, 0] = (p @ v).reshape(-1, dim)
            if case["op"] == "weigh":
                after[b, :, :n] = s["before"][layer, b, :, :n].double() + p.sum(1)
        out.append(a if case["op"] == "attn" else (a, after) if case["op"] == "weigh" else (a, new_k, new_v))
    return out
