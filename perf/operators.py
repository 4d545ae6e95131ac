"""The quantised KV cache and the decode attention that reads it: what is measured.

The cache holds each key and value vector of 64 channels as two blocks of 32
channels. A block is one power-of-two scale (a byte) and 32 elements of 4 bits
(sign, 2 exponent bits, 1 mantissa bit) or 8 bits (sign, 4, 3). Three passes:

* ``kv``: keys and values of new tokens are quantised into the cache, then
  read back as bf16 (``kv_quant.write``, ``kv_quant.read``);
* ``attn``: one query token per row attends the first ``used[b]`` positions of
  its row (``flash_decode.QuantFlashDecode``), ``used`` 0 giving zeros;
* ``fused``: the decode layer's form. The packed QKV projection arrives as fp32
  partials; they are summed and rounded to bf16, rotated, the new token's key
  and value are quantised into the cache, and the query attends the row with
  them (``QuantFlashDecode.fused_qkv``). The new token's key and value are
  read back beside the attention.

Heads, rows and contexts are those of the two configuration presets (24 or 16
query heads over 8 KV heads) and of the attention tests (1 to 8 query heads per
KV head), one user to 128 rows, contexts to 4096, and generic long contexts.
Decode cases run several layers, each with a cache of its own, as a model's
step does.
"""
import functools
import math

import numpy as np
import torch

own = False

DEVICE = "cuda:0"
BF16 = torch.bfloat16
D = 64
THETA = 10000.0


def listed():
    return [
        # The store of one decode step of the headline batch: 64 tokens, one per row; latency counts.
        dict(name="kv_store_b64_4bit", op="kv", bits=4, kv_heads=8, rows=64, low=1, high=1),
        # One ordinary prompt of 700 tokens into the 8-bit cache and back.
        dict(name="kv_prompt_700_8bit", op="kv", bits=8, kv_heads=8, rows=1, low=700, high=700),
        # A packed prefill of 48 ragged prompts (about 50,000 tokens).
        dict(name="kv_prefill_48_ragged_4bit", op="kv", bits=4, kv_heads=8, rows=48, low=64, high=2048),
        # One user of the small model in a short chat.
        dict(name="attn_b1_512_4bit", op="attn", bits=4, kv_heads=8, groups=2, layers=4, rows=1, low=509, high=509),
        # The headline decode: 64 rows in their second thousand of tokens.
        dict(name="attn_b64_4bit", op="attn", bits=4, kv_heads=8, groups=3, layers=4, rows=64, low=1025, high=1279),
        # Few users with long contexts: the key range has to be split to fill the GPU.
        dict(name="attn_b3_long_8bit", op="attn", bits=8, kv_heads=8, groups=2, layers=4, rows=3, low=2049, high=4001),
        # Long-context serving: the largest batch over ragged contexts, bound by the KV stream.
        dict(name="attn_b128_ragged_4bit", op="attn", bits=4, kv_heads=8, groups=3, layers=2, rows=128, low=1024,
             high=4095),
        # A few documents of up to 32768 tokens.
        dict(name="attn_b8_32768_4bit", op="attn", bits=4, kv_heads=8, groups=3, layers=1, rows=8, low=8191,
             high=32768),
        # The decode layer of one user: reduction, rotation, store and attention in one launch.
        dict(name="fused_b1_1000_4bit", op="fused", bits=4, kv_heads=8, groups=3, layers=4, rows=1, low=1000,
             high=1000),
        # The small model's batch of 32 after prompts of 512 tokens, 8 bits.
        dict(name="fused_b32_8bit", op="fused", bits=8, kv_heads=8, groups=2, layers=4, rows=32, low=513, high=640),
        # The headline decode layer.
        dict(name="fused_b64_4bit", op="fused", bits=4, kv_heads=8, groups=3, layers=4, rows=64, low=1025, high=1279),
        # The largest batch over ragged contexts, 8 bits.
        dict(name="fused_b128_ragged_8bit", op="fused", bits=8, kv_heads=8, groups=3, layers=2, rows=128, low=1024,
             high=4095),
    ]


def _log_int(rng, low, high):
    return min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1))) - 0.5)) or low)


def draw(rng):
    op = rng.choice(["kv", "attn", "attn", "fused"])
    case = dict(op=op, bits=rng.choice([4, 4, 8]), kv_heads=rng.choice([1, 2, 8, 8]))
    if op == "kv":
        rows = _log_int(rng, 1, 128)
        high = _log_int(rng, 1, min(4095, 65536 // rows))
        case.update(rows=rows, low=max(1, int(high * rng.uniform(0.1, 1.0))), high=high)
        return case
    rows = _log_int(rng, 1, 128)
    high = _log_int(rng, 1, min(32768, 524288 // rows))
    low = int(high * rng.uniform(0.1, 1.0))
    if op == "fused":
        low = max(1, low)           # the new token is attended, so a row holds one at least
    elif rng.random() < 0.3:
        low = 0                     # rows that hold nothing yet
    case.update(groups=rng.choice([1, 2, 2, 3, 3, 4, 6, 8]), layers=1 if rows * high > 65536 else rng.randint(1, 4),
                rows=rows, low=low, high=high)
    return case


# ---------------------------------------------------------------- inputs --

def _lengths(case):
    return np.rint(np.linspace(case["low"], case["high"], case["rows"])).astype(np.int64)


def _capacity(longest):
    return -(-longest // 256) * 256


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


def _table(capacity):
    """RoPE's ``[capacity, 64]``: cos | sin, bf16."""
    inv = THETA ** (-torch.arange(0, D, 2, device=DEVICE).double() / D)
    angle = torch.arange(capacity, device=DEVICE).double()[:, None] * inv
    return torch.cat((angle.cos(), angle.sin()), -1).to(BF16)


# A 4-bit element's 8 magnitudes in the order of its codes; an 8-bit element's 128 (the last is no number).
_E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
_E4M3 = ([m * 2.0 ** -9 for m in range(8)]
         + [(1 + (c & 7) / 8) * 2.0 ** ((c >> 3) - 7) for c in range(8, 127)] + [math.nan])


@functools.lru_cache(None)
def _values(bits):
    """The value of every code, sign bit on top, fp32."""
    magnitudes = _E2M1 if bits == 4 else _E4M3
    return torch.tensor(magnitudes + [-m for m in magnitudes], device=DEVICE)


@functools.lru_cache(None)
def _scales():
    """The value of every scale byte: 2^(b - 127); 0 stands for zero and 255 for no number."""
    return torch.tensor([0.0] + [2.0 ** (b - 127) for b in range(1, 255)] + [math.nan], device=DEVICE)


def _exponents(x, bits):
    """Blocks ``x [..., 32]`` in fp32: the exponent of each, the smallest e with max|x| <= T 2^e."""
    m, e = torch.frexp(x.abs().amax(-1))
    return (e - 3 + (m > 0.875)).clamp(-126, 125) if bits == 4 else (e - 9 + (m > 0.90625)).clamp(-126, 119)


def _elements(x, e, bits):
    """The blocks' elements in units of 2^e: rounded to the type's grid (ties to even), held to its largest value."""
    a = torch.ldexp(x, -e[..., None])
    least, mantissa, most = (0, 1, 6.0) if bits == 4 else (-6, 3, 448.0)
    step = torch.exp2(((torch.frexp(a)[1] - 1).clamp(min=least) - mantissa).float())
    return (torch.round(a / step) * step).clamp(-most, most)


def _pack(x, bits):
    """Vectors ``x [..., 64]`` as the cache holds them: codes ``[..., 8 * bits]`` and scale bytes ``[..., 2]``."""
    blocks = x.float().unflatten(-1, (2, 32))
    e = _exponents(blocks, bits)
    value = _elements(blocks, e, bits).flatten(-2)
    magnitudes = _values(bits)[:8 if bits == 4 else 127]
    code = torch.bucketize(value.abs(), magnitudes).to(torch.uint8) | (torch.signbit(value).to(torch.uint8) << (bits - 1))
    if bits == 4:
        code = code[..., 0::2] | (code[..., 1::2] << 4)
    return code, (e + 127).to(torch.uint8)


def _history(inp, case):
    """A cache of random keys and values, one layer after the other: codes and scale bytes (k0, k1, v0, v1)."""
    shape = (case["layers"], case["rows"], case["kv_heads"], _capacity(case["high"]))
    k, v = (torch.empty(*shape, 8 * case["bits"], device=DEVICE, dtype=torch.uint8) for _ in range(2))
    scales = torch.empty(*shape, 4, device=DEVICE, dtype=torch.uint8)
    for layer in range(shape[0]):
        for row in range(0, shape[1], 8):
            for side, at in ((k, 0), (v, 2)):
                codes, s = _pack(inp.vectors(min(8, shape[1] - row), *shape[2:], D), case["bits"])
                side[layer, row:row + 8] = codes
                scales[layer, row:row + 8, ..., at:at + 2] = s
    return k, v, scales


def prepare(case, seed):
    inp = _Inputs(seed)
    lengths = inp.lengths(case)
    if case["op"] == "kv":
        # packed tokens as a prefill's QKV projection leaves them: K and V heads are columns of one row
        tokens, heads = int(lengths.sum()), case["kv_heads"]
        qkv = inp.vectors(tokens, 2 * heads, D)
        positions = torch.from_numpy(np.concatenate([np.arange(n) for n in lengths])).to(DEVICE)
        slots = torch.from_numpy(np.repeat(np.arange(case["rows"]), lengths)).to(DEVICE)
        if case["high"] == 1:       # a decode step's tokens lie anywhere in their rows
            positions = torch.from_numpy(inp.rng.randint(0, 1280, tokens)).to(DEVICE)
        return dict(case=case, k=qkv[:, :heads, None], v=qkv[:, heads:, None], positions=positions, slots=slots,
                    active=torch.ones(tokens, dtype=torch.bool, device=DEVICE),
                    capacity=_capacity(1280 if case["high"] == 1 else case["high"]))
    k, v, scales = _history(inp, case)
    used = torch.from_numpy(lengths).to(DEVICE, torch.int32)
    s = dict(case=case, k=k, v=v, scales=scales, used=used, scale=1.0 / math.sqrt(D))
    hq, hkv = case["kv_heads"] * case["groups"], case["kv_heads"]
    if case["op"] == "attn":
        s["q"] = [(1.5 * inp.normal(case["rows"], hq, 1, D)).to(BF16) for _ in range(case["layers"])]
    else:
        # three K slices of the packed projection; query columns larger, so that scores spread as a trained model's do
        size = torch.ones((hq + 2 * hkv) * D, device=DEVICE)
        size[:hq * D] = 1.5
        s["partials"] = [inp.normal(3, case["rows"], size.numel(), std=3 ** -0.5) * size for _ in range(case["layers"])]
        s["positions"] = used.long() - 1
        s["table"] = _table(k.shape[3])
        # a ragged batch's rows are dispatched longest first, as the engine has it
        ragged = case["high"] > 1.25 * case["low"]
        s["order"] = torch.argsort(used, descending=True, stable=True).int() if ragged else None
    return s


# ------------------------------------------------------- the framework's --

def _own_cache(s):
    from litemoe_amd.cache import QuantKVCache
    if "cache" not in s:
        case = s["case"]
        if case["op"] == "kv":
            shape = (1, case["rows"], case["kv_heads"], s["capacity"])
            s["cache"] = QuantKVCache.empty(*shape, DEVICE, bits=case["bits"])
        else:
            s["cache"] = QuantKVCache.over(s["k"], s["v"], s["scales"])
    return s["cache"]


def _own_flash(s):
    from litemoe_amd.flash_decode import QuantFlashDecode
    if "flash" not in s:
        case = s["case"]
        s["flash"] = QuantFlashDecode(case["rows"], case["kv_heads"], case["groups"], s["k"].shape[3], DEVICE,
                                      max(1, case["high"]), bits=case["bits"])
    return s["flash"]


def _own_run(s):
    from litemoe_amd import kv_quant
    case, cache = s["case"], _own_cache(s)
    if case["op"] == "kv":
        kv_quant.write(cache, 0, s["k"], s["v"], s["positions"], s["active"], s["slots"])
        return kv_quant.read(cache, 0, s["positions"], s["slots"])
    flash, out = _own_flash(s), []
    for layer in range(case["layers"]):
        held = cache.layer(layer)
        if case["op"] == "attn":
            out.append(flash(s["q"][layer], *held, None, None, s["scale"], used=s["used"]))
        else:
            a = flash.fused_qkv(s["partials"][layer], s["table"], s["positions"], None, *held, s["scale"], s["used"],
                                case["kv_heads"] * case["groups"], row_order=s["order"])
            out.append((a, *kv_quant.read(cache, layer, s["positions"], cache.slots)))
    return out


# ----------------------------------------------------------- plain forms --

def _unpack(codes, scales, bits):
    """What codes ``[..., 8 * bits]`` and scale bytes ``[..., 2]`` stand for: ``[..., 64]`` in fp32."""
    if bits == 4:
        codes = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    return (_values(bits)[codes.int()].unflatten(-1, (2, 32)) * _scales()[scales.int()][..., None]).flatten(-2)


def _attend(q, k, v, used, scale):
    """``q [B, H, G, 64]`` over ``k, v [B, H, C, 64]`` in fp32; a row with nothing used gives zeros."""
    seen = torch.arange(k.shape[2], device=DEVICE)[None] < used[:, None]
    scores = (torch.matmul(q, k.transpose(-1, -2)) * scale).masked_fill(~seen[:, None, None], -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True).clamp(min=-1e30))
    return torch.matmul(p, v) / p.sum(-1, keepdim=True).clamp(min=1e-30)


def _rotate(x, cos, sin):
    """Neox rotation in bf16: each product and each sum is rounded, as the operator is defined."""
    x1, x2 = x[..., :D // 2], x[..., D // 2:]
    return torch.cat((x1 * cos - x2 * sin, x2 * cos + x1 * sin), -1)


def _plain_run(s):
    case, bits = s["case"], s["case"]["bits"]
    if case["op"] == "kv":
        if "cache" not in s:
            shape = (case["rows"], case["kv_heads"], s["capacity"])
            s["cache"] = [torch.zeros(*shape, n, device=DEVICE, dtype=torch.uint8) for n in (8 * bits, 2) * 2]
        back = []
        for x, (codes, scales) in ((s["k"], s["cache"][:2]), (s["v"], s["cache"][2:])):
            at = (s["slots"], slice(None), s["positions"])
            codes[at], scales[at] = _pack(x[:, :, 0], bits)
            back.append(_unpack(codes[at], scales[at], bits).to(BF16)[:, :, None])
        return tuple(back)
    rows, hkv, groups = case["rows"], case["kv_heads"], case["groups"]
    out = []
    for layer in range(case["layers"]):
        ck, cv, cs = s["k"][layer], s["v"][layer], s["scales"][layer]
        if case["op"] == "attn":
            q = s["q"][layer].view(rows, hkv, groups, D)
        else:
            p = s["partials"][layer]
            qkv = ((p[0] + p[1]) + p[2]).to(BF16).view(rows, -1, D)
            cos, sin = s["table"][s["positions"]][:, None].chunk(2, -1)
            q = _rotate(qkv[:, :hkv * groups], cos, sin).view(rows, hkv, groups, D)
            k, v = _rotate(qkv[:, hkv * groups:-hkv], cos, sin), qkv[:, -hkv:]
            at = (torch.arange(rows, device=DEVICE), slice(None), s["positions"])
            for x, side, part in ((k, ck, slice(0, 2)), (v, cv, slice(2, 4))):
                side[at], cs[at + (part,)] = _pack(x, bits)
        a = _attend(q.float(), _unpack(ck, cs[..., :2], bits), _unpack(cv, cs[..., 2:], bits), s["used"], s["scale"])
        a = a.to(BF16).view(rows, hkv * groups, 1, D)
        if case["op"] == "fused":
            a = (a, *(_unpack(side[at], cs[at + (part,)], bits).to(BF16)[:, :, None]
                      for side, part in ((ck, slice(0, 2)), (cv, slice(2, 4)))))
        out.append(a)
    return out


def run(state):
    return _own_run(state) if own else _plain_run(state)


# ------------------------------------------------------- work and 64 bits --

def work(case):
    token = case["kv_heads"] * (16 * case["bits"] + 4)    # K and V codes and scale bytes of one position
    total, rows = int(_lengths(case).sum()), case["rows"]
    if case["op"] == "kv":
        # written: bf16 in, codes out; read back: codes in, bf16 out; a position, slot (and mask) a token each time
        return dict(bytes=total * 2 * (token + case["kv_heads"] * 256 + 16), flops=total * case["kv_heads"] * 256)
    hq = case["kv_heads"] * case["groups"]
    if case["op"] == "attn":
        size, flops = total * token + rows * (hq * 256 + 4), total * hq * 256
    else:
        new = rows * (token + case["kv_heads"] * 256)     # stored, and read back as bf16
        size = total * token + rows * ((hq + 2 * case["kv_heads"]) * 768 + hq * 128 + 140) + new
        flops = total * hq * 256 + rows * (hq + 2 * case["kv_heads"]) * 512
    return dict(bytes=case["layers"] * size, flops=case["layers"] * flops)


def _quantised64(x, bits):
    """Vectors ``[..., 64]`` in 64 bits as their quantised values: the nearest of the type's values under each scale."""
    t, grid = (7.0, _E2M1) if bits == 4 else (464.0, _E4M3[:127])
    blocks = x.double().reshape(-1, 32)
    e = torch.full((blocks.shape[0],), -126.0, dtype=torch.float64, device=DEVICE)
    most = blocks.abs().max(-1).values
    guess = torch.floor(torch.log2(most.clamp(min=2.0 ** -140) / t)) - 1
    for _ in range(3):              # up to the smallest exponent that covers the block
        guess = torch.where(most > t * 2.0 ** guess, guess + 1, guess)
    e = torch.maximum(e, guess).clamp(max=125 if bits == 4 else 119)[:, None]
    grid = torch.tensor(grid, dtype=torch.float64, device=DEVICE)
    a = (blocks / 2.0 ** e).abs().contiguous()
    above = torch.searchsorted(grid, a).clamp(1, len(grid) - 1)
    down, up = a - grid[above - 1], grid[above] - a
    nearest = torch.where((up < down) | ((up == down) & (above % 2 == 0)), above, above - 1)
    return (torch.sign(blocks) * grid[nearest] * 2.0 ** e).view(x.shape)


def _rotate64(x, cos, sin):
    def held(t):                    # the operator's own bf16 results
        return t.to(BF16).double()
    half = D // 2
    return torch.cat((held(held(x[..., :half] * cos) - held(x[..., half:] * sin)),
                      held(held(x[..., half:] * cos) + held(x[..., :half] * sin))), -1)


def _decoded64(codes, scales, bits):
    """Codes of one row back to numbers from the bit fields themselves, in 64 bits."""
    c = codes.long()
    if bits == 4:
        c = torch.stack((c % 16, c // 16), -1).reshape(*c.shape[:-1], D)
        sign, field, m = c // 8, c // 2 % 4, (c % 2).double() / 2
        value = torch.where(field > 0, (1 + m) * 2.0 ** (field - 1).double(), m)
    else:
        sign, field, m = c // 128, c // 8 % 16, (c % 8).double() / 8
        value = torch.where(field > 0, (1 + m) * 2.0 ** (field - 7).double(), m * 2.0 ** -6)
    scale = 2.0 ** (scales.double() - 127)
    return (1 - 2 * sign) * value * scale.repeat_interleave(32, -1)


def exact(case, seed):
    s, bits = prepare(case, seed), case["bits"]
    if case["op"] == "kv":
        return tuple(_quantised64(s[side], bits) for side in ("k", "v"))
    rows, hkv, groups = case["rows"], case["kv_heads"], case["groups"]
    out = []
    for layer in range(case["layers"]):
        a = torch.zeros(rows, hkv * groups, 1, D, dtype=torch.float64, device=DEVICE)
        new_k, new_v = (torch.zeros(rows, hkv, 1, D, dtype=torch.float64, device=DEVICE) for _ in range(2))
        for b, n in enumerate(s["used"].tolist()):
            if case["op"] == "attn":
                q = s["q"][layer][b].double().view(hkv, groups, D)
            else:
                heads = s["partials"][layer][:, b].double().sum(0).to(BF16).double().view(-1, D)
                cos, sin = s["table"][n - 1].double().split(D // 2)
                q = _rotate64(heads[:hkv * groups], cos, sin).view(hkv, groups, D)
                new_k[b, :, 0] = _quantised64(_rotate64(heads[hkv * groups:-hkv], cos, sin), bits)
                new_v[b, :, 0] = _quantised64(heads[-hkv:], bits)
            if not n:
                continue
            k = _decoded64(s["k"][layer, b, :, :n], s["scales"][layer, b, :, :n, :2], bits)
            v = _decoded64(s["v"][layer, b, :, :n], s["scales"][layer, b, :, :n, 2:], bits)
            if case["op"] == "fused":
                k[:, n - 1], v[:, n - 1] = new_k[b, :, 0], new_v[b, :, 0]
            a[b, :, 0] = (torch.softmax(q @ k.transpose(1, 2) * s["scale"], -1) @ v).reshape(-1, D)
        out.append(a if case["op"] == "attn" else (a, new_k, new_v))
    return out
