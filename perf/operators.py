"""What the 4-bit key/value cache's speed is measured on: writing it, reading it back, and attention over it.

A cache page holds runs of *units*: 16 tokens of one kv head, ``D + D / 8`` bytes a token.  Sixteen neighbouring
features of a token's key or value share a scale: a value is ``scale * code``, the code one of the 4-bit
numbers 0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign, the scale an unsigned byte of 5 exponent and 3 mantissa bits (the
bits 7 to 14 of the 16-bit float of the same value).  A unit is ``[key codes | value codes | key scales | value
scales]``; :func:`unpacked` says where each of them lies.

Kinds
-----
store       raw ``[q | k | v]`` projection rows of new tokens: q and k normed per head and rotated, keys and values
            into the 4-bit pages; then the pages that hold the new tokens read back
decode      one token a request attends to its request's pages
prompt      portions of prompts attend to their requests' pages, the portions' own keys included

``listed()`` holds the cases by name, ``draw()`` gives others of the same ranges.  Sizes are the layer shapes and
contexts that this repository's benchmark and tests use.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda:0"
EPS = 1e-6
THETA = 1e6
UNIT = 16           # tokens a unit
GROUP = 16          # features that share a scale
MAX_SCALE = 10240.0
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
MOST_KEYS = 64 * 6200           # keys of all requests of the largest decode case
MOST_PAIRS = 14_500_000         # (token, visible key) pairs of the largest prompt case


def listed():
    return [
        # one user's chat: the smallest write, where latency counts
        {"name": "store_one", "kind": "store", "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128, "page": 16, "requests": 1, "tokens": 1,
         "depth": 1023},
        # a busy server: 64 requests write a token each, pages of 64 keys
        {"name": "store_batch", "kind": "store", "heads": 64, "kv_heads": 8, "dim": 128, "rotary": 128, "page": 64, "requests": 64, "tokens": 64,
         "depth": 1100},
        # the headline prompt goes into the cache
        {"name": "store_prompt", "kind": "store", "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128, "page": 16, "requests": 1, "tokens": 2048,
         "depth": 0},
        # three ragged portions of a model with small heads, part of each rotated
        {"name": "store_ragged", "kind": "store", "heads": 12, "kv_heads": 4, "dim": 64, "rotary": 32, "page": 32, "requests": 3, "tokens": 1337,
         "depth": 501},
        # one user's chat: the smallest attention, where latency counts
        {"name": "decode_one", "kind": "decode", "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "requests": 1, "depth": 1024, "window": 0},
        # the headline batch
        {"name": "decode_eight", "kind": "decode", "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "requests": 8, "depth": 1024, "window": 0},
        # a busy server with long conversations
        {"name": "decode_many", "kind": "decode", "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "requests": 64, "depth": 8192, "window": 0},
        # few requests over very long documents, eight query heads a kv head
        {"name": "decode_long", "kind": "decode", "heads": 64, "kv_heads": 8, "dim": 128, "page": 64, "requests": 3, "depth": 32768, "window": 0},
        # small heads under a sliding window, an odd number of requests
        {"name": "decode_window", "kind": "decode", "heads": 12, "kv_heads": 4, "dim": 64, "page": 32, "requests": 37, "depth": 2900, "window": 1000},
        # the headline prompt
        {"name": "prompt_whole", "kind": "prompt", "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "requests": 1, "tokens": 2048, "depth": 0,
         "window": 0},
        # a late portion of a long prompt
        {"name": "prompt_late", "kind": "prompt", "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "requests": 1, "tokens": 1531, "depth": 9000,
         "window": 0},
        # a few tokens that three users add to their conversations
        {"name": "prompt_short", "kind": "prompt", "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "requests": 3, "tokens": 19, "depth": 2100,
         "window": 0},
    ]


def _between(rng, low, high):
    """Spread over the logarithm."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["store", "decode", "decode", "prompt"])
    heads, kv_heads, dim = rng.choice([(32, 8, 128), (64, 8, 128), (12, 4, 64), (16, 16, 128), (32, 2, 128), (20, 4, 64), (8, 1, 128)])
    case = {"kind": kind, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": rng.choice([16, 16, 32, 48, 64])}
    if kind == "store":
        case["rotary"] = rng.choice([dim, dim, dim // 2, 20, 0])
        case["tokens"] = _between(rng, 1, 2000)
        case["requests"] = rng.choice([1, rng.randint(1, min(case["tokens"], 64)), case["tokens"] if case["tokens"] <= 64 else 3])
        case["depth"] = rng.choice([0, _between(rng, 1, 5000)])
        return case
    if kind == "decode":
        case["requests"] = _between(rng, 1, 64)
        case["depth"] = _between(rng, 1, min(32000, MOST_KEYS // case["requests"] * 8 // max(8, kv_heads)))
        case["window"] = rng.choice([0, 0, 0, _between(rng, 1, 4000)])
        return case
    case["requests"] = rng.randint(1, 4)
    case["tokens"] = _between(rng, 2 * case["requests"], 1500)
    room = MOST_PAIRS * 32 // heads // case["tokens"] - case["tokens"] // case["requests"] - 1
    case["depth"] = rng.choice([0, min(_between(rng, 20, 9000), max(0, room))])
    case["window"] = rng.choice([0, 0, _between(rng, 1, 3000)])
    return case


# ------------------------------------------------------------------ sizes of a case
def lengths(case):
    """(new tokens, tokens held before them) of every request; a decoding request's token is among its ``depth``."""
    n = case["requests"]
    spread = lambda i: case["depth"] - i * (case["depth"] // 2) // n
    if case["kind"] == "decode":
        return [(1, max(1, spread(i)) - 1) for i in range(n)]
    base, more = divmod(case["tokens"], n)
    cut = [base + (i < more) for i in range(n)]
    for i in range(0, n - 1, 2):                    # ragged: neighbours give and take a third
        third = cut[i + 1] // 3
        cut[i], cut[i + 1] = cut[i] + third, cut[i + 1] - third
    return [(cut[i], spread(i)) for i in range(n)]


def first_visible(position, window):
    return max(0, position - window + 1) if window else 0


def unit_bytes(dim):
    return UNIT * (dim + dim // 8)


def touched(case):
    """Pages that hold a new token, over all requests."""
    page = case["page"]
    return sum((held + new - 1) // page - held // page + 1 for new, held in lengths(case))


def work(case):
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    token_bytes = d + d // 8                        # a token's key and value of one kv head
    if case["kind"] == "store":
        t = case["tokens"]
        back = touched(case) * case["page"] * kv
        moved = t * (2 * h + 2 * kv) * d * 2 + t * kv * token_bytes + t * case["rotary"] * 4 + 2 * d * 4 + back * (token_bytes + 4 * d)
        return {"bytes": moved, "flops": t * (h + kv) * d * 8 + t * kv * d * 2 * 4 + back * 2 * d}
    pairs = keys = 0
    for new, held in lengths(case):
        end = held + new
        keys += end - first_visible(held, case["window"])
        if case["window"]:
            w = case["window"]
            pairs += sum(min(w, p + 1) for p in range(held, end))
        else:
            pairs += (held + 1 + end) * new // 2
    rows = sum(new for new, _ in lengths(case))
    return {"bytes": rows * h * d * 2 * 2 + keys * kv * token_bytes, "flops": 4 * h * d * pairs}


# ------------------------------------------------------------------ the format, in elementary operations
def _scales(largest):
    """The scale of groups whose largest magnitude is ``largest`` (float64): nearest, ties to even."""
    wanted = (largest / 6.0).clamp(max=MAX_SCALE)
    exponent = torch.frexp(wanted).exponent - 1
    step = torch.ldexp(torch.ones_like(wanted), exponent.clamp(min=-14) - 3)
    return (torch.round(wanted / step) * step).clamp(max=MAX_SCALE)


def quantised(x):
    """(codes, scale bytes) of float64 rows [.., features]: uint8 [.., features] and [.., features / 16]."""
    groups = x.unflatten(-1, (-1, GROUP))
    scale = _scales(groups.abs().amax(-1))
    at = groups.abs() / torch.where(scale > 0, scale, torch.ones_like(scale)).unsqueeze(-1)
    at = torch.where(scale.unsqueeze(-1) > 0, at, torch.zeros_like(at))
    code = ((at > 0.25).to(torch.uint8) + (at >= 0.75) + (at > 1.25) + (at >= 1.75) + (at > 2.5) + (at >= 3.5) + (at > 5.0))
    code = code + (groups < 0).to(torch.uint8) * 8
    return code.flatten(-2), (scale.to(torch.float16).view(torch.int16) >> 7).to(torch.uint8)


def places(dim, device):
    """Where in a unit the codes of a token's key and value and their scales lie: four index tensors [16, ..]
    (two features a byte, the even one in the low half).

    The order is that in which the 32 lanes ``4 g + t`` of a warp hold them in a product of 16 x 8 x 16: the keys by rows;
    of the values lane ``4 g + t`` holds features ``D / 8 * g ..`` of tokens ``2 t, 2 t + 1`` and then of ``2 t + 8,
    2 t + 9``.  Key scales: lane ``4 g + t`` holds those of features ``D / 4 * t ..`` of tokens ``g`` and ``g + 8``."""
    r = torch.arange(UNIT, device=device).view(-1, 1)
    p, s = torch.arange(dim // 2, device=device), torch.arange(dim // GROUP, device=device)
    half, t, odd = r >> 3, (r >> 1) & 3, r & 1
    piece = dim // 16
    k_code = r * (dim // 2) + p
    v_code = UNIT * dim // 2 + half * (4 * dim) + ((p // piece * 4 + t) * 2 + odd) * piece + p % piece
    per = dim // 64
    k_scale = UNIT * dim + ((r & 7) * 4 + s // per) * (2 * per) + half * per + s % per
    v_scale = UNIT * (dim + dim // 16) + (s * 4 + t) * 4 + half * 2 + odd
    return k_code, v_code, k_scale, v_scale


def packed(k, v):
    """Units [n, kv heads, bytes] of float64 rows [n, kv heads, 16, dim]."""
    n, kv, _, dim = k.shape
    out = torch.zeros((n, kv, unit_bytes(dim)), dtype=torch.uint8, device=k.device)
    k_code, v_code, k_scale, v_scale = places(dim, k.device)
    kc, ks = quantised(k)
    vc, vs = quantised(v)
    out[:, :, k_code] = kc[..., 0::2] | (kc[..., 1::2] << 4)
    out[:, :, v_code] = vc[..., 0::2] | (vc[..., 1::2] << 4)
    out[:, :, k_scale], out[:, :, v_scale] = ks, vs
    return out


def unpacked(units, dim):
    """Float32 keys and values [.., 16, dim] of units [.., bytes]."""
    lead = units.shape[:-1]
    level = torch.tensor(LEVELS + tuple(-v for v in LEVELS), dtype=torch.float32, device=units.device)
    piece = dim // 16
    k_code = units[..., :UNIT * dim // 2].reshape(*lead, UNIT, dim // 2)
    v_code = units[..., UNIT * dim // 2:UNIT * dim].reshape(*lead, 2, 8, 4, 2, piece)       # half, lane row, pair, odd, bytes
    v_code = v_code.movedim(-4, -2).reshape(*lead, UNIT, dim // 2)
    scales = (units[..., UNIT * dim:].to(torch.int16) << 7).view(torch.float16).float()
    ks = scales[..., :dim].reshape(*lead, 8, 4, 2, dim // 64).movedim(-2, -4).reshape(*lead, UNIT, dim // GROUP)
    vs = scales[..., dim:].reshape(*lead, dim // GROUP, 4, 2, 2).movedim(-4, -1).movedim(-4, -3).reshape(*lead, UNIT, dim // GROUP)

    def values(code, scale):
        pair = torch.stack([code & 15, code >> 4], dim=-1).flatten(-2).int()
        return (level[pair].unflatten(-1, (-1, GROUP)) * scale.unsqueeze(-1)).flatten(-2)

    return values(k_code, ks), values(v_code, vs)


# ------------------------------------------------------------------ inputs
def _pages_of(case, g):
    """Block tables [requests, blocks] over a pool of shuffled pages, -1 behind a request's last page, and the pool's size."""
    page = case["page"]
    counts = [-(-(new + held) // page) for new, held in lengths(case)]
    order = torch.randperm(sum(counts) + 3, generator=g, device=DEV).int()
    table = torch.full((len(counts), max(counts)), -1, dtype=torch.int32, device=DEV)
    at = 0
    for i, n in enumerate(counts):
        table[i, :n] = order[at:at + n]
        at += n
    return table, order.numel()


def _rows(case):
    """Per new token: its position and its request, and the segments (request, first row, tokens, first position)."""
    positions, request, segments, at = [], [], [], 0
    for i, (new, held) in enumerate(lengths(case)):
        positions += range(held, held + new)
        request += [i] * new
        segments.append((i, at, new, held))
        at += new
    as_ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    return as_ints(positions), as_ints(request), segments


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    h, kv, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    normal = lambda *shape: torch.randn(shape, generator=g, device=DEV, dtype=torch.float32)
    table, pages = _pages_of(case, g)
    positions, request, segments = _rows(case)
    tokens = positions.numel()
    s = {"case": case, "table": table, "positions": positions, "request": request, "segments": segments,
         "ends": torch.tensor([held + new for new, held in lengths(case)], dtype=torch.int32, device=DEV),
         "firsts": torch.tensor([at for _, at, _, _ in segments] + [tokens], dtype=torch.int32, device=DEV),
         "requests": torch.arange(len(segments), dtype=torch.int32, device=DEV),
         "max_end": max(held + new for new, held in lengths(case))}
    # keys as a norm and a rotation leave them, a few features larger than the others; values of about one
    loud = 1.0 + 3.0 * (torch.rand((kv, 1, d), generator=g, device=DEV) > 0.96)
    units = pages * page // UNIT
    cache = torch.empty((units, kv, unit_bytes(d)), dtype=torch.uint8, device=DEV)
    for at in range(0, units, 2048):
        n = min(2048, units - at)
        cache[at:at + n] = packed((normal(n, kv, UNIT, d) * loud).double(), normal(n, kv, UNIT, d).double())
    s["cache"] = cache.view(pages, page // UNIT, kv, -1).transpose(1, 2).contiguous()
    if case["kind"] == "store":
        s["qkv"] = normal(tokens, (h + 2 * kv) * d).bfloat16()
        s["q_weight"], s["k_weight"] = 1.0 + 0.1 * normal(d), 1.0 + 0.1 * normal(d)
        block = table[request.long(), (positions // page).long()]
        s["slots"] = block * page + positions % page
        s["touched"] = torch.unique(block)
        s["rot"] = None
        if case["rotary"]:
            half = case["rotary"] // 2
            angle = positions.double().unsqueeze(1) * THETA ** (torch.arange(half, device=DEV, dtype=torch.float64) / -half)
            s["rot"] = torch.stack([angle.cos(), angle.sin()], dim=-1).float()
    else:
        s["q"] = (1.5 * normal(tokens, h * d)).bfloat16()
    return s


# ------------------------------------------------------------------ one pass
def run(state):
    kind = state["case"]["kind"]
    if kind == "store":
        return _store_own(state) if own else _store(state)
    return _attention_own(state) if own else _attention(state)


def _rotated(x, rot):
    if rot is None:
        return x
    half = rot.shape[1]
    c, s = rot[:, None, :, 0].to(x.dtype), rot[:, None, :, 1].to(x.dtype)
    a, b, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
    return torch.cat([a * c - b * s, b * c + a * s, rest], dim=-1)


def _store(s):
    case = s["case"]
    h, kv, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    tokens = s["positions"].numel()
    x = s["qkv"].view(tokens, h + 2 * kv, d)
    normed = lambda y, w: y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * w
    q = _rotated(normed(x[:, :h].float(), s["q_weight"]), s["rot"])
    # which side of a border a key falls on is told in 64 bits
    k = _rotated(normed(x[:, h:h + kv].double(), s["k_weight"].double()), s["rot"])
    kc, ks = quantised(k)
    vc, vs = quantised(x[:, h + kv:].double())
    slots = s["slots"].long()
    at, r = (slots // page, slots % page // UNIT), slots % UNIT
    cache = s["cache"]
    k_code, v_code, k_scale, v_scale = (p[r].unsqueeze(1) for p in places(d, cache.device))
    page_at, unit_at = at[0].view(-1, 1, 1), at[1].view(-1, 1, 1)
    head_at = torch.arange(kv, device=cache.device).view(1, -1, 1)
    cache[page_at, head_at, unit_at, k_code] = kc[..., 0::2] | (kc[..., 1::2] << 4)
    cache[page_at, head_at, unit_at, v_code] = vc[..., 0::2] | (vc[..., 1::2] << 4)
    cache[page_at, head_at, unit_at, k_scale] = ks
    cache[page_at, head_at, unit_at, v_scale] = vs
    back = [v.flatten(2, 3).bfloat16() for v in unpacked(cache[s["touched"].long()], d)]
    return {"q": q.reshape(tokens, h * d).bfloat16(), "k": back[0], "v": back[1]}


def _attention(s):
    case = s["case"]
    h, kv, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    n, window = len(s["segments"]), case["window"]
    held = s["table"] >= 0
    k, v = unpacked(s["cache"][s["table"].clamp(min=0).long()], d)       # [requests, blocks, kv heads, units, 16, dim]
    k, v = (x.transpose(1, 2).reshape(n, kv, -1, d) for x in (k, v))
    # the requests' tokens side by side, rows that a request does not have left out again at the end
    most = max(new for _, _, new, _ in s["segments"])
    row = s["firsts"][:-1].view(-1, 1).long() + torch.arange(most, device=DEV)
    real = row < s["firsts"][1:].view(-1, 1)
    row = torch.where(real, row, torch.zeros_like(row))
    q = s["q"].float()[row].view(n, most, kv, h // kv, d).permute(0, 2, 3, 1, 4)
    position = s["positions"][row].view(n, 1, 1, most, 1)
    key = torch.arange(k.shape[2], device=DEV)
    seen = (key <= position) & held.repeat_interleave(page, dim=1).view(n, 1, 1, 1, -1)
    if window:
        seen = seen & (key > position - window)
    score = q.reshape(n, kv, -1, d) @ k.transpose(2, 3) * d ** -0.5
    score = score.view(n, kv, h // kv, most, -1).masked_fill_(~seen, -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    out = (p.view(n, kv, -1, p.shape[-1]) @ v).view(n, kv, h // kv, most, d) / p.sum(-1, keepdim=True)
    return out.permute(0, 3, 1, 2, 4).reshape(n, most, h * d)[real].bfloat16()


_staging = []       # the program's pinned buffers


def _store_own(s):
    from mrun_b200.kernels import ops
    case = s["case"]
    q = s["qkv"].new_empty((s["qkv"].shape[0], case["heads"] * case["dim"]))
    ops.qk_norm_rope_cache_fp4(s["qkv"], case["heads"], case["kv_heads"], case["dim"], s["q_weight"], s["k_weight"], EPS, s["rot"],
                               case["rotary"], s["slots"], s["cache"], q_out=q)
    k, v = ops.fp4_pages(s["cache"], case["dim"], s["touched"])
    return {"q": q, "k": k, "v": v}


def _attention_own(s):
    from mrun_b200.engine.batch import GroupView, HostStaging, SegmentInfo, StepContext
    from mrun_b200.kernels.attention import paged_attention_fp4
    if not _staging:
        _staging.append(HostStaging(torch.device(DEV)))
    case = s["case"]
    tokens = s["positions"].numel()
    group = GroupView(s["table"], None, s["table"].shape[1])
    ctx = StepContext(num_tokens=tokens, num_segments=len(s["segments"]), segments=[SegmentInfo(i, at, new, held) for i, at, new, held in s["segments"]],
                      token_ids=None, positions=s["positions"], token_slot=s["request"], seg_q_start=s["firsts"], seg_kv_len=s["ends"],
                      seg_slot=s["requests"], groups={}, max_q_len=max(new for _, _, new, _ in s["segments"]), max_kv_len=s["max_end"],
                      page_size=case["page"], real_tokens=tokens, upload=_staging[0].upload)
    out = torch.empty_like(s["q"])
    return paged_attention_fp4(s["q"], s["q"].shape[1], out, s["cache"], group, ctx, case["heads"], case["dim"], case["dim"] ** -0.5, case["window"])


# ------------------------------------------------------------------ the same in 64 bits, from the definitions
def _exact_held(x):
    """What groups of 16 of float64 ``x`` are held as: the nearest scale of the table, then the nearest level."""
    table = (torch.arange(256, dtype=torch.int16) << 7).view(torch.float16).double()
    table = table[table <= MAX_SCALE].to(x.device)                       # ascending; a byte is its index
    groups = x.reshape(*x.shape[:-1], -1, GROUP)
    wanted = (groups.abs().amax(-1) / 6.0).clamp(max=MAX_SCALE).contiguous()
    above = torch.searchsorted(table, wanted).clamp(1, table.numel() - 1)
    low, high = table[above - 1], table[above]
    up = (wanted - low > high - wanted) | ((wanted - low == high - wanted) & (above % 2 == 0))
    scale = torch.where(up, high, low).unsqueeze(-1)
    order = [0, 2, 4, 6, 1, 3, 5, 7]                                     # the first of two equally near ones is even
    level = torch.tensor([LEVELS[i] for i in order], dtype=torch.float64, device=x.device)
    near = (groups.abs().unsqueeze(-1) - level * scale.unsqueeze(-1)).abs().argmin(-1)
    return (torch.copysign(level[near], groups) * scale).reshape(x.shape)


def _exact_unit(units, dim):
    """Float64 keys and values [n, 16, dim] of units [n, bytes], byte by byte from where each value lies."""
    table = torch.tensor(LEVELS, dtype=torch.float64, device=units.device)
    token, feature = torch.meshgrid(torch.arange(UNIT, device=units.device), torch.arange(dim, device=units.device), indexing="ij")
    half, pair, odd, lane = token // 8, token // 2 % 4, token % 2, dim // 8
    code_at = {"k": token * (dim // 2) + feature // 2,
               "v": 8 * dim + half * 4 * dim + (feature // lane * 8 + pair * 2 + odd) * (dim // 16) + feature % lane // 2}
    scale_at = {"k": 16 * dim + (token % 8 * 4 + feature // (dim // 4)) * (dim // 32) + half * (dim // 64) + feature % (dim // 4) // 16,
                "v": 17 * dim + feature // 16 * 16 + pair * 4 + half * 2 + odd}
    out = []
    for name in "kv":
        byte = units[:, code_at[name]].long()
        nibble = torch.where(feature % 2 == 0, byte % 16, byte // 16)
        exponent, mantissa = units[:, scale_at[name]].long() // 8, units[:, scale_at[name]].long() % 8
        scale = torch.where(exponent > 0, (8 + mantissa) * 2.0 ** (exponent.double() - 18), mantissa * 2.0 ** -17)
        out.append(table[nibble % 8] * (1 - 2 * (nibble // 8)) * scale)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    h, kv, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    cache = s["cache"]
    if case["kind"] == "store":
        x = s["qkv"].double().reshape(-1, h + 2 * kv, d)
        parts = {}
        for name, part, weight in (("q", x[:, :h], s["q_weight"]), ("k", x[:, h:h + kv], s["k_weight"])):
            y = part / torch.sqrt((part * part).sum(-1, keepdim=True) / d + EPS) * weight.double()
            if s["rot"] is not None:
                half = case["rotary"] // 2
                turn = torch.view_as_complex(s["rot"].double()).unsqueeze(1)
                z = torch.complex(y[..., :half].contiguous(), y[..., half:2 * half].contiguous()) * turn
                y = torch.cat([z.real, z.imag, y[..., 2 * half:]], dim=-1)
            parts[name] = y
        out = {}
        old = [v.reshape(-1, kv, page, d) for v in _exact_unit(cache[s["touched"].long()].reshape(-1, unit_bytes(d)), d)]
        where = torch.searchsorted(s["touched"], s["slots"] // page)
        for name, rows, before in (("k", parts["k"], old[0]), ("v", x[:, h + kv:], old[1])):
            for at in range(0, rows.shape[0], 256):
                before[where[at:at + 256].long(), :, (s["slots"][at:at + 256] % page).long()] = _exact_held(rows[at:at + 256])
            out[name] = before
        return {"q": parts["q"].reshape(-1, h * d), "k": out["k"], "v": out["v"]}
    out = torch.empty((s["positions"].numel(), h, d), dtype=torch.float64, device=DEV)
    q = s["q"].double().view(-1, h, d)
    for request, at, new, held in s["segments"]:
        end = held + new
        blocks = s["table"][request, :-(-end // page)].long()
        for head in range(kv):
            k, v = (x.reshape(-1, d)[:end] for x in _exact_unit(cache[blocks, head].reshape(-1, unit_bytes(d)), d))
            key = torch.arange(end, device=DEV).view(1, -1)
            for first in range(0, new, 512):
                last = min(new, first + 512)
                position = torch.arange(held + first, held + last, device=DEV).view(-1, 1)
                hidden = key > position
                if case["window"]:
                    hidden = hidden | (key <= position - case["window"])
                mine = slice(head * (h // kv), (head + 1) * (h // kv))
                score = torch.einsum("qhd,kd->hqk", q[at + first:at + last, mine], k) / math.sqrt(d)
                share = torch.softmax(score.masked_fill(hidden, -math.inf), dim=-1)
                out[at + first:at + last, mine] = torch.einsum("hqk,kd->qhd", share, v)
    return out.reshape(-1, h * d)
