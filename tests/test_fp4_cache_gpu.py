"""The kernels of the 4-bit key/value cache against 64-bit arithmetic: what is written, read back, and attended to.

Tolerances.  A held value is a scale times a code: what is read back equals the definition's value bit for bit, and the
cache's bytes are the definition's.  A norm and a rotation in 32 bits are within 2^-19 of a q's value relative to its head's largest
(sixteen roundings), far inside the half step 2^-9 (relative: 2^-8) of its bfloat16 rounding: 1.01 * 2^-8 of the value plus 2^-19 of
the largest.  Attention: P is rounded to 16-bit floats (2^-11 relative, and absolutely 2^-25 / 32 of the row's maximum for the smallest), the
exponential is within 2^-21, sums are in 32 bits, the output is rounded to bfloat16 (2^-8 of its value): an output is off by at most
2^-8 |o| + 2^-10 sum p |v|, and sum p |v| is at most the largest |v|.  Prompt portions go through the kernels over bfloat16 pages, which round P to
bfloat16: 2^-8 |o| + 2^-7 max |v|.
"""
import math

import pytest
import torch

import plain_fp4

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def ops():
    from mrun_b200.kernels import ops as module
    return module


def rotated(x, rot):
    """x float64 [tokens, heads, dim], rot [tokens, pairs, 2] or None."""
    if rot is None:
        return x
    c, s = rot.double()[:, None, :, 0], rot.double()[:, None, :, 1]
    n = c.shape[-1]
    a, b = x[..., :n], x[..., n:2 * n]
    return torch.cat([a * c - b * s, b * c + a * s, x[..., 2 * n:]], -1)


def normed(x, weight, eps):
    if weight is None:
        return x
    return x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * weight.double()


def inputs(tokens, heads, kv_heads, dim, rotary, seed, norm=True):
    g = torch.Generator().manual_seed(seed)
    normal = lambda *shape: torch.randn(shape, generator=g)
    qkv = (normal(tokens, (heads + 2 * kv_heads) * dim) * torch.exp(normal(tokens, 1))).bfloat16()
    weights = (1 + 0.2 * normal(dim), 1 + 0.2 * normal(dim)) if norm else (None, None)
    rot = None
    if rotary:
        angle = torch.randint(0, 5000, (tokens, 1), generator=g).double() * 1e4 ** (-torch.arange(rotary // 2).double() / (rotary // 2))
        rot = torch.stack([angle.cos(), angle.sin()], -1).float()
    return qkv, weights, rot


def to(t):
    return None if t is None else t.to(DEV)


@pytest.mark.parametrize("heads, kv_heads, dim, rotary, page, tokens, norm", [
    (4, 2, 128, 128, 16, 1, True), (32, 8, 128, 128, 16, 37, True), (5, 5, 64, 64, 32, 19, True), (6, 1, 128, 64, 48, 33, True),
    (3, 3, 64, 20, 16, 21, True), (2, 1, 128, 2, 64, 5, True), (7, 1, 64, 0, 16, 18, True), (4, 2, 128, 0, 16, 40, False),
    (4, 4, 64, 62, 16, 9, False), (1, 1, 128, 126, 32, 64, True)])
def test_write_and_read_back(heads, kv_heads, dim, rotary, page, tokens, norm):
    qkv, (qw, kw), rot = inputs(tokens, heads, kv_heads, dim, rotary, seed=tokens, norm=norm)
    pages, eps = 2 + tokens // page, 1e-5
    g = torch.Generator().manual_seed(7)
    slots = torch.randperm(pages * page, generator=g)[:tokens].int()
    if tokens > 4:
        slots[2], slots[4] = -1, pages * page + 3           # written nowhere
    x = qkv.double().view(tokens, heads + 2 * kv_heads, dim)
    q_want = rotated(normed(x[:, :heads], qw, eps), rot)
    k_want = plain_fp4.held(rotated(normed(x[:, heads:heads + kv_heads], kw, eps), rot))
    v_want = plain_fp4.held(x[:, heads + kv_heads:])
    cache = torch.zeros(ops().fp4_cache_shape(pages, kv_heads, page, dim), dtype=torch.uint8, device=DEV)

    wide = torch.full((tokens, heads * dim + 24), 7.0, dtype=torch.bfloat16, device=DEV)
    given = qkv.to(DEV)
    q = ops().qk_norm_rope_cache_fp4(given, heads, kv_heads, dim, to(qw), to(kw), eps, to(rot), rotary, slots.to(DEV), cache,
                                     q_out=wide[:, :heads * dim])
    assert torch.equal(given.cpu(), qkv) and (wide[:, heads * dim:] == 7).all()
    again = torch.zeros_like(cache)
    in_place = ops().qk_norm_rope_cache_fp4(given, heads, kv_heads, dim, to(qw), to(kw), eps, to(rot), rotary, slots.to(DEV), again)
    assert torch.equal(in_place, q) and torch.equal(again, cache) and torch.equal(given[:, :heads * dim], q)
    assert torch.equal(given[:, heads * dim:].cpu(), qkv[:, heads * dim:])

    off = (q.double().cpu().view_as(q_want) - q_want).abs()
    assert (off <= 1.01 * 2.0 ** -8 * q_want.abs() + 2.0 ** -19 * q_want.abs().amax(-1, keepdim=True)).all()

    # the bytes, token by token: the codes and scales of the definition where it says they lie, and nothing else
    want = torch.zeros(cache.shape, dtype=torch.int64)
    value = {}
    for i, slot in enumerate(slots.tolist()):
        if not 0 <= slot < pages * page:
            continue
        at, r = (slot // page, slice(None), slot % page // 16), slot % 16
        value[slot] = (k_want[0][i], v_want[0][i])
        for is_v, (_, code, byte) in ((False, k_want), (True, v_want)):
            for f in range(dim):
                want[at + (plain_fp4.code_at(dim, r, f, is_v),)] |= code[i, :, f] << 4 * (f % 2)
            for s in range(dim // 16):
                want[at + (plain_fp4.scale_at(dim, r, s, is_v),)] = byte[i, :, s]
    assert torch.equal(cache.cpu().long(), want)

    order = torch.cat([torch.randperm(pages, generator=g).int(), torch.tensor([-1, pages, 0], dtype=torch.int32)])
    k, v = ops().fp4_pages(cache, dim, order.to(DEV))
    k, v = k.double().cpu(), v.double().cpu()
    assert k.shape == (pages + 3, kv_heads, page, dim)
    for i, p in enumerate(order.tolist()):
        for offset in range(page):
            kk, vv = value.get(p * page + offset, (torch.zeros(kv_heads, dim).double(),) * 2) if 0 <= p < pages else (torch.zeros(kv_heads, dim).double(),) * 2
            assert torch.equal(k[i, :, offset], kk) and torch.equal(v[i, :, offset], vv)


@pytest.mark.parametrize("heads, kv_heads, dim, rotary, tokens, norm", [
    (32, 8, 128, 128, 357, True), (12, 4, 64, 32, 1337, True), (5, 3, 64, 64, 3001, True), (1, 1, 64, 0, 66001, False),
    (4, 1, 128, 0, 9001, True), (20, 4, 128, 96, 8003, True), (1, 3, 128, 64, 12001, False)])
def test_write_of_many_tokens(heads, kv_heads, dim, rotary, tokens, norm):
    """Steps of so many heads that lanes take several of a token: what the same tokens give in steps of few."""
    qkv, (qw, kw), rot = inputs(tokens, heads, kv_heads, dim, rotary, seed=tokens, norm=norm)
    qw, kw, rot, qkv = to(qw), to(kw), to(rot), qkv.to(DEV)
    page, eps = 32, 1e-6
    pages = tokens // page + 1
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(1))[:tokens].int()
    slots[::7], slots[3::50] = -1, pages * page
    slots = slots.to(DEV)
    caches = [torch.zeros(ops().fp4_cache_shape(pages, kv_heads, page, dim), dtype=torch.uint8, device=DEV) for _ in range(3)]
    write = lambda x, t0, t1, cache, **kw_: ops().qk_norm_rope_cache_fp4(
        x[t0:t1], heads, kv_heads, dim, qw, kw, eps, rot if rot is None else rot[t0:t1], rotary, slots[t0:t1], cache, **kw_)
    q = torch.empty(tokens, heads * dim, dtype=torch.bfloat16, device=DEV)
    write(qkv, 0, tokens, caches[0], q_out=q)
    few = 16384 // (heads + 2 * kv_heads)
    apart = torch.empty_like(q)
    for t0 in range(0, tokens, few):
        write(qkv, t0, min(t0 + few, tokens), caches[1], q_out=apart[t0:t0 + few])
    given = qkv.clone()
    in_place = write(given, 0, tokens, caches[2])
    assert torch.equal(q, apart) and torch.equal(in_place, q) and torch.equal(given[:, heads * dim:], qkv[:, heads * dim:])
    assert torch.equal(caches[0], caches[1]) and torch.equal(caches[0], caches[2]) and caches[0].any()


def test_values_on_borders_and_beyond():
    """Ties of codes and of scales, groups of zeros, tiny, huge and infinite values, and NaN."""
    dim, kv_heads, page = 64, 1, 16
    v = torch.zeros(16, dim)
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0])
    for i in range(8):
        v[0, 8 * i:8 * i + 8] = ties * 2.0 ** (i - 4) * (-1) ** i
    v[1, :16] = 6 * 17 / 16                                    # a scale half-way between two bytes: to the even one
    v[1, 16:32] = 6 * 19 / 16
    v[1, 32:48] = 6 * 2.0 ** -18                              # half of the least scale
    v[1, 48:] = 6 * 2.0 ** -17 * 1.5
    v[2, :16], v[2, 16:32], v[2, 32:48], v[2, 48:] = 1e-30, 3e38, 61440.0, 7e4
    v[3, 5], v[3, 20], v[3, 40] = math.inf, -math.inf, math.nan
    v[4] = torch.linspace(-1e-4, 1e-4, dim)
    v[5] = torch.linspace(-3e-5, 3e-5, dim)                    # below the least normal scale
    v[6, ::3] = -0.0
    g = torch.Generator().manual_seed(3)
    v[7:] = torch.randn(9, dim, generator=g) * torch.exp(4 * torch.randn(9, dim, generator=g))
    v = v.bfloat16()
    qkv = torch.cat([v, v, v], 1)                              # without weights and rotation a key is held as it is
    cache = torch.zeros(ops().fp4_cache_shape(1, kv_heads, page, dim), dtype=torch.uint8, device=DEV)
    ops().qk_norm_rope_cache_fp4(qkv.to(DEV), 1, kv_heads, dim, None, None, 0.0, None, 0, torch.arange(16, dtype=torch.int32, device=DEV), cache)
    got = ops().fp4_pages(cache, dim, torch.zeros(1, dtype=torch.int32, device=DEV))
    want = plain_fp4.held(v.double())[0]
    for x in got:
        assert torch.equal(torch.nan_to_num(x[0, 0].double().cpu(), nan=12345.0), torch.nan_to_num(want, nan=12345.0))
    assert torch.isnan(want).sum() == 48 and (want[1, :16] == 6).all() and (want[1, 16:32] == 7.5).all() and (want[1, 32:48] == 0).all()


@pytest.mark.parametrize("rotary", [0, 64])
def test_keys_far_from_one(rotary):
    """Rows whose sum of squares leaves the range of 32 bits at either end, without and with an eps, rows with zeros, one value that
    outweighs all others, a NaN and an infinity: the codes of the formula, which the 32-bit sums cannot tell."""
    dim, heads = 64, 3
    g = torch.Generator().manual_seed(2)
    x = torch.randn(12, dim, generator=g).double()
    x *= 10.0 ** torch.tensor([30, 20, 18.5, 8, 0, -8, -14, -17, -20, -30, -37, 0]).double().view(-1, 1)
    x[4, ::2] = 0
    x[11, 7] = 1e6
    x = x.bfloat16()
    bad = torch.randn(2, dim, generator=g).bfloat16()
    bad[0, 3], bad[1, 40] = math.nan, math.inf
    k = torch.cat([x, bad])
    tokens = k.shape[0]
    qkv = torch.cat([torch.zeros(tokens, dim, dtype=torch.bfloat16), k, torch.zeros(tokens, dim, dtype=torch.bfloat16)], 1)
    weight = 1 + 0.2 * torch.randn(dim, generator=g)
    rot = None
    if rotary:
        angle = torch.rand(tokens, rotary // 2, generator=g).double() * 6
        rot = torch.stack([angle.cos(), angle.sin()], -1).float()
    for eps in (0.0, 1e-6, 1e-19):
        cache = torch.zeros(ops().fp4_cache_shape(1, 1, 16, dim), dtype=torch.uint8, device=DEV)
        ops().qk_norm_rope_cache_fp4(qkv.to(DEV), 1, 1, dim, weight.to(DEV), weight.to(DEV), eps, to(rot), rotary,
                                     torch.arange(tokens, dtype=torch.int32, device=DEV), cache)
        got = ops().fp4_pages(cache, dim, torch.zeros(1, dtype=torch.int32, device=DEV))[0][0, 0, :tokens].double().cpu()
        y = rotated(normed(k.double().view(tokens, 1, dim), weight, float(torch.tensor(eps, dtype=torch.float32))), rot)
        want = plain_fp4.held(y)[0].view(tokens, dim)
        assert torch.equal(got[:12], want[:12]) and torch.isnan(got[12]).all() and torch.equal(torch.isnan(got[13]), torch.isnan(want[13]))


def test_calls_on_two_streams_at_once():
    heads, kv_heads, dim, page = 32, 8, 128, 16
    lengths = [3000, 20, 1999, 640]
    c = Filled(lengths, kv_heads, dim, page, seed=8)
    table = c.table.to(DEV)
    steps = [step_of([(j, 1, n - 1 - 3 * i) for j, n in enumerate(lengths)], table, page) for i in range(2)]
    q = [c.queries(4, heads, dim).to(DEV) for _ in range(2)]
    out = [[torch.zeros_like(q[0]) for _ in range(20)] for _ in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for turn in range(20):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                attention(q[i], heads * dim, out[i][turn], c.cache, steps[i][1], steps[i][0], heads, dim, dim ** -0.5)
    torch.cuda.synchronize()
    for i in range(2):
        want = torch.stack([plain_fp4.attend(q[i][j:j + 1].cpu().view(1, heads, dim), c.k[j], c.v[j], [n - 1 - 3 * i], dim ** -0.5).view(-1)
                            for j, n in enumerate(lengths)])
        close(out[i][0], want, c.v, 2.0 ** -10)
        assert all(torch.equal(out[i][0], x) for x in out[i])


def step_of(segments, table, page, tokens=None):
    """A step over segments (slot, tokens, first position), with padding rows up to ``tokens``."""
    from mrun_b200.engine.batch import GroupView, HostStaging, SegmentInfo, StepContext
    infos, positions, slots = [], [], []
    for slot, n, first in segments:
        infos.append(SegmentInfo(slot, len(positions), n, first))
        positions += range(first, first + n)
        slots += [slot] * n
    real = len(positions)
    pad = (tokens or real) - real
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    staging = HostStaging(torch.device(DEV))
    ctx = StepContext(num_tokens=real + pad, num_segments=len(infos), segments=infos, token_ids=None, positions=ints(positions + [-1] * pad),
                      token_slot=ints(slots + [0] * pad), seg_q_start=None, seg_kv_len=None, seg_slot=None, groups={},
                      max_q_len=max(n for _, n, _ in segments), max_kv_len=max(n + first for _, n, first in segments), page_size=page,
                      real_tokens=real, upload=staging.upload)
    return ctx, GroupView(table, None, table.shape[1])


class Filled:
    """Requests of given lengths in a 4-bit cache of random values, built from the definition; unused places hold bytes that would
    be NaN."""

    def __init__(self, lengths, kv_heads, dim, page, seed=0, spare=3, extra_blocks=0):
        g = torch.Generator().manual_seed(seed)
        blocks = [-(-n // page) for n in lengths]
        pages = sum(blocks) + spare
        order = torch.randperm(pages, generator=g).tolist()
        self.table = torch.full((len(lengths), max(blocks) + extra_blocks), -1, dtype=torch.int32)
        self.k, self.v = [], []
        cache = torch.full((pages, kv_heads, page // 16, 18 * dim), 255, dtype=torch.uint8)
        for i, n in enumerate(lengths):
            k, v = (torch.randn(n, kv_heads, dim, generator=g).double() * torch.exp(0.5 * torch.randn(n, kv_heads, 1, generator=g)) for _ in range(2))
            self.k.append(plain_fp4.held(k)[0]); self.v.append(plain_fp4.held(v)[0])
            whole = -(-n // 16) * 16
            padded = [torch.cat([x, torch.full((whole - n, kv_heads, dim), math.nan, dtype=torch.float64)]).view(whole // 16, 16, kv_heads, dim).transpose(1, 2)
                      for x in (k, v)]
            units = plain_fp4.units_of(*padded)                # [units, kv heads, bytes]
            for b in range(blocks[i]):
                p = order.pop()
                self.table[i, b] = p
                part = units[b * page // 16:(b + 1) * page // 16]
                cache[p, :, :part.shape[0]] = part.transpose(0, 1)
        self.cache = cache.to(DEV)
        self.g = g

    def queries(self, tokens, heads, dim):
        return torch.randn(tokens, heads * dim, generator=self.g).bfloat16()


def close(got, want, v, p_step):
    """Within the bounds above."""
    most = max(float(x.abs().nan_to_num().max()) for x in v)
    off = (got.double().cpu() - want).abs()
    bound = 1.01 * 2.0 ** -8 * want.abs() + p_step * most
    assert torch.isfinite(got).all() and (off <= bound).all(), float((off - bound).max())


def attention(*args, **kw):
    from mrun_b200.kernels.attention import paged_attention_fp4
    return paged_attention_fp4(*args, **kw)


@pytest.mark.parametrize("heads, kv_heads, dim, page, lengths, window", [
    (4, 1, 128, 16, [1], 0), (4, 1, 128, 16, [16, 17], 0), (32, 8, 128, 16, [63, 64, 65, 200], 0), (8, 8, 64, 32, [33, 5, 300], 0),
    (12, 4, 64, 48, [97, 1, 700, 350], 100), (16, 1, 128, 64, [1000, 130], 0), (40, 2, 128, 16, [260, 31], 0), (34, 2, 64, 16, [77, 400], 33),
    (7, 7, 128, 32, [513], 1), (8, 1, 128, 16, [500, 90, 64], -64), (6, 2, 64, 16, [3000], 0), (9, 1, 64, 16, [1500, 40], 0)])
def test_single_tokens(heads, kv_heads, dim, page, lengths, window):
    c = Filled(lengths, kv_heads, dim, page, seed=len(lengths) + heads)
    q = c.queries(len(lengths) + 2, heads, dim)
    ctx, group = step_of([(i, 1, n - 1) for i, n in enumerate(lengths)], c.table.to(DEV), page, tokens=len(lengths) + 2)
    out = torch.full((len(lengths) + 2, heads * dim), 3.0, dtype=torch.bfloat16, device=DEV)
    wide = torch.zeros(len(lengths) + 2, heads * dim + 8, dtype=torch.bfloat16, device=DEV)
    wide[:, :heads * dim] = q.to(DEV)
    attention(wide, wide.shape[1], out, c.cache, group, ctx, heads, dim, dim ** -0.5, window)
    assert (out[len(lengths):] == 0).all()
    want = torch.stack([plain_fp4.attend(q[i:i + 1].view(1, heads, dim), c.k[i], c.v[i], [n - 1], dim ** -0.5, window)[0].reshape(-1)
                        for i, n in enumerate(lengths)])
    close(out[:len(lengths)], want, c.v, 2.0 ** -10)


@pytest.mark.parametrize("tiles", [0, 1, 2, 1 << 20])
@pytest.mark.parametrize("heads, kv_heads, dim, lengths, window", [
    (8, 2, 128, [1, 900, 129, 2500], 0), (16, 1, 64, [128, 700, 5000], 0), (5, 1, 128, [3000, 60], 1000), (32, 8, 128, [2000], 0)])
def test_pairs_in_clusters_and_dealt_to_all_blocks(monkeypatch, tiles, heads, kv_heads, dim, lengths, window):
    """The same steps with a cluster a pair (of 8 blocks to one, some without a tile) and with the tiles of all pairs dealt to all blocks."""
    from mrun_b200.kernels import attention as module
    rule = module.fp4_cluster
    assert [rule(8, 592, keys) for keys in (1, 256, 257, 513, 1025, 4096, 4097)] == [1, 1, 2, 4, 8, 8, 0]
    assert [rule(pairs, 592, 2048) for pairs in (74, 75, 148, 149, 296, 297)] == [8, 4, 4, 2, 2, 1]
    assert [rule(pairs, 592, 2049) for pairs in (296, 297, 2048)] == [0, 0, 0] and rule(2048, 592, 2048) == 1 and rule(65536, 592, 1) == 0
    monkeypatch.setattr(module, "FP4_CLUSTER_TILES", (tiles,) * 3)
    page = 16
    c = Filled(lengths, kv_heads, dim, page, seed=heads)
    repeat = 1 + tiles % 2 * 20                                # also with so many pairs that clusters are smaller
    tokens = repeat * len(lengths) + 1
    q = c.queries(tokens, heads, dim)
    segments = [(i, 1, n - 1) for _ in range(repeat) for i, n in enumerate(lengths)]
    ctx, group = step_of(segments, c.table.to(DEV), page, tokens=tokens)
    out = torch.full((tokens, heads * dim), 3.0, dtype=torch.bfloat16, device=DEV)
    attention(q.to(DEV), heads * dim, out, c.cache, group, ctx, heads, dim, dim ** -0.5, window)
    want = torch.cat([plain_fp4.attend(q[t:t + 1].view(1, heads, dim), c.k[i], c.v[i], [pos], dim ** -0.5, window).view(1, -1)
                      for t, (i, _, pos) in enumerate(segments)])
    assert (out[-1] == 0).all()
    close(out[:-1], want, c.v, 2.0 ** -10)


def test_spans_that_do_not_fit_are_refused():
    c = Filled([100], 2, 64, 16)
    table = torch.zeros(1, 2, dtype=torch.int32, device=DEV)
    rows = torch.zeros(8, dtype=torch.int32, device=DEV)
    for span in ((0, 0, 100, 0, -1, 4), (0, 0, 100, 0, 5, 4), (0, 0, 100, 0, 0, -1), (0, -64, 36, 0, 0, 4), (0, 0, 300, 0, 0, 4), (0, 0, 100, 1, 0, 4),
                 (0, 64, 64, 0, 0, 4), (0, 0, 100, -1, 0, 4), (0, 1 << 32, (1 << 32) + 50, 0, 0, 4), (0, 128, 228, 0, 0, 4)):
        with pytest.raises(ops().KernelError):
            ops().fp4_spans(c.cache, 64, c.table.to(DEV), [span], 2, 64, table, rows)
    assert not table.any() and not rows.any()


def test_pages_far_behind_the_first_bytes():
    """A cache of more than 2^32 bytes: writing, reading back, and attention of both kinds in its last pages, as in a small one."""
    heads, kv_heads, dim, page, n = 16, 8, 128, 32, 700
    shape = ops().fp4_cache_shape(130_000, kv_heads, page, dim)
    blocks = -(-n // page)
    assert math.prod(shape) > 2 ** 32
    qkv, (qw, kw), rot = inputs(n, heads, kv_heads, dim, dim, seed=3)
    got = []
    for pages in (blocks, shape[0]):
        cache = torch.empty((pages,) + shape[1:], dtype=torch.uint8, device=DEV)
        first = pages - blocks
        slots = (torch.arange(n, dtype=torch.int32) + first * page).to(DEV)
        table = torch.arange(first, pages, dtype=torch.int32, device=DEV).view(1, -1)
        q = ops().qk_norm_rope_cache_fp4(qkv.to(DEV), heads, kv_heads, dim, to(qw), to(kw), 1e-6, to(rot), dim, slots, cache)
        back = ops().fp4_pages(cache, dim, table[0])
        outs = []
        for segments in ([(0, n, 0)], [(0, 1, t) for t in range(0, n, 9)]):
            ctx, group = step_of(segments, table, page)
            out = torch.empty(ctx.num_tokens, heads * dim, dtype=torch.bfloat16, device=DEV)
            rows = q if len(segments) == 1 else q[::9]
            attention(rows.contiguous(), heads * dim, out, cache, group, ctx, heads, dim, dim ** -0.5)
            outs.append(out)
        got.append([q.clone(), *(x.reshape(blocks, kv_heads, page, dim).transpose(1, 2).reshape(-1, kv_heads, dim)[:n] for x in back), *outs])
        del cache
    for a, b in zip(*got):
        assert torch.equal(a, b) and torch.isfinite(a).all()


def test_more_heads_than_a_grid_of_clusters_takes():
    heads, dim, page, tokens = 256, 64, 16, 256
    c = Filled([40], heads, dim, page, seed=5)
    q = c.queries(tokens, heads, dim)
    ctx, group = step_of([(0, 1, t % 40) for t in range(tokens)], c.table.to(DEV), page)
    out = torch.empty(tokens, heads * dim, dtype=torch.bfloat16, device=DEV)
    attention(q.to(DEV), heads * dim, out, c.cache, group, ctx, heads, dim, 0.1)
    rows = list(range(0, tokens, 37)) + [tokens - 1]
    want = torch.cat([plain_fp4.attend(q[t:t + 1].view(1, heads, dim), c.k[0], c.v[0], [t % 40], 0.1).view(1, -1) for t in rows])
    close(out[rows], want, c.v, 2.0 ** -10)


def test_many_tokens_of_a_launch_and_more():
    """More tokens than a launch takes, many of them of the same request, with rows of padding between them."""
    heads, kv_heads, dim, page = 4, 2, 64, 16
    lengths = [150, 40, 300]
    c = Filled(lengths, kv_heads, dim, page, seed=4)
    g = torch.Generator().manual_seed(1)
    tokens = 1100
    slot = torch.randint(0, 3, (tokens,), generator=g)
    position = (torch.rand(tokens, generator=g) * torch.tensor(lengths)[slot]).int()
    position[torch.rand(tokens, generator=g) < 0.1] = -1
    q = c.queries(tokens, heads, dim)
    ctx, group = step_of([(0, 1, 0)] * tokens, c.table.to(DEV), page)
    ctx.positions, ctx.token_slot, ctx.max_kv_len = position.to(DEV), slot.int().to(DEV), 300
    out = torch.full((tokens, heads * dim), 3.0, dtype=torch.bfloat16, device=DEV)
    attention(q.to(DEV), heads * dim, out, c.cache, group, ctx, heads, dim, 0.2, 0)
    want = torch.cat([plain_fp4.attend(q[i:i + 1].view(1, heads, dim), c.k[s], c.v[s], [p], 0.2).view(1, -1)
                      for i, (s, p) in enumerate(zip(slot.tolist(), position.tolist()))])
    close(out, want, c.v, 2.0 ** -10)


def test_pages_that_are_not_held():
    """A freed page, a page number outside the cache, a table that is too short, a request outside the table; a request without any."""
    heads, kv_heads, dim, page = 8, 2, 128, 16
    c = Filled([200, 90, 50, 64], kv_heads, dim, page, seed=2)
    table = c.table.clone()
    table[0, 3] = -1
    table[0, 5] = 10 ** 6
    table[2] = -1
    seen = torch.ones(200, dtype=torch.bool)
    seen[48:64] = seen[80:96] = False
    segments = [(0, 1, 199), (1, 1, 2000), (2, 1, 49), (3, 1, 63), (9, 1, 30), (-4, 1, 30)]
    ctx, group = step_of(segments, table.to(DEV), page)
    q = c.queries(6, heads, dim)
    out = torch.full((6, heads * dim), 3.0, dtype=torch.bfloat16, device=DEV)
    attention(q.to(DEV), heads * dim, out, c.cache, group, ctx, heads, dim, dim ** -0.5)
    at = lambda i, s, pos, seen=None: plain_fp4.attend(q[i:i + 1].view(1, heads, dim), c.k[s], c.v[s], [pos], dim ** -0.5, 0, seen).view(-1)
    assert (out[[2, 4, 5]] == 0).all()
    # the second request's position lies behind what its table holds: its last page is read to its end, where NaN lie
    assert torch.isnan(out[1]).any()
    close(out[[0, 3]], torch.stack([at(0, 0, 199, seen), at(3, 3, 63)]), c.v, 2.0 ** -10)


def test_large_and_small_magnitudes():
    """Queries whose product with a half would overflow, tiny ones, a head of zeros; values at the ends of the format's range."""
    heads, kv_heads, dim, page, n = 8, 1, 64, 16, 120
    c = Filled([n], kv_heads, dim, page, seed=9)
    g = torch.Generator().manual_seed(5)
    size = torch.exp(3 * torch.randn(n, 1, 1, generator=g)).double() * 3e-4
    v = torch.randn(n, 1, dim, generator=g).double() * size
    v[:3] = v[:3] / v[:3].abs().max() * 6e4
    k = torch.randn(n, 1, dim, generator=g).double()
    pad = lambda x: torch.cat([x, torch.zeros(8, 1, dim, dtype=torch.float64)]).view(8, 16, 1, dim).transpose(1, 2)
    units = plain_fp4.units_of(pad(k), pad(v))
    for b in range(8):
        c.cache[int(c.table[0, b]), :, 0] = units[b].to(DEV)
    k, v = plain_fp4.held(k)[0], plain_fp4.held(v)[0]
    q = torch.randn(heads, dim, generator=g).double() * 10.0 ** torch.tensor([30, 8, 0, -3, -20, -38, 0, 4]).view(-1, 1)
    q[6] = 0
    q = q.bfloat16()
    for scale in (0.125, 1e-9, 1e-29):
        ctx, group = step_of([(0, 1, n - 1)], c.table.to(DEV), page)
        out = torch.empty(1, heads * dim, dtype=torch.bfloat16, device=DEV)
        attention(q.view(1, -1).to(DEV), heads * dim, out, c.cache, group, ctx, heads, dim, scale)
        want = plain_fp4.attend(q.view(1, heads, dim), k, v, [n - 1], scale).view(1, -1)
        close(out, want, [v], 2.0 ** -10)


def test_nan_where_it_is_seen_and_only_there():
    heads, kv_heads, dim, page, n = 4, 1, 128, 16, 100
    c = Filled([n], kv_heads, dim, page, seed=3)
    unit = c.cache[int(c.table[0, 3]), 0, 0]                  # tokens 48 .. 63
    unit[plain_fp4.scale_at(dim, 2, 1, True)] = 255          # features 16 .. 31 of the value of token 50
    q = c.queries(3, heads, dim)
    ctx, group = step_of([(0, 1, 49), (0, 1, 50), (0, 1, 99)], c.table.to(DEV), page)
    out = torch.empty(3, heads * dim, dtype=torch.bfloat16, device=DEV)
    attention(q.to(DEV), heads * dim, out, c.cache, group, ctx, heads, dim, dim ** -0.5)
    rows = out.view(3, heads, dim)
    assert torch.isfinite(rows[0]).all()
    assert torch.isnan(rows[1:, :, 16:32]).all() and torch.isfinite(rows[1:, :, :16]).all() and torch.isfinite(rows[1:, :, 32:]).all()
    attention(q.to(DEV), heads * dim, out, c.cache, group, ctx, heads, dim, dim ** -0.5, 20)
    assert torch.isfinite(rows[2]).all()                       # the window has passed token 50


@pytest.mark.parametrize("heads, kv_heads, dim, page, segments, window", [
    (8, 2, 128, 16, [(70, 0)], 0), (8, 2, 128, 16, [(5, 130), (1, 60), (300, 33), (4, 9)], 0), (12, 4, 64, 48, [(33, 500), (6, 1)], 100),
    (4, 4, 64, 32, [(129, 0), (1, 0), (2, 300)], 0), (32, 2, 128, 64, [(50, 700)], 256), (68, 1, 64, 16, [(9, 40), (3, 2)], 0),
    (16, 2, 128, 16, [(130, 127), (7, 257)], -128)])
def test_prompt_portions(heads, kv_heads, dim, page, segments, window):
    lengths = [n + held for n, held in segments]
    c = Filled(lengths, kv_heads, dim, page, seed=heads)
    tokens = sum(n for n, _ in segments)
    q = c.queries(tokens + 3, heads, dim)
    ctx, group = step_of([(i, n, held) for i, (n, held) in enumerate(segments)], c.table.to(DEV), page, tokens=tokens + 3)
    out = torch.full((tokens + 3, heads * dim), 3.0, dtype=torch.bfloat16, device=DEV)
    attention(q.to(DEV), heads * dim, out, c.cache, group, ctx, heads, dim, dim ** -0.5, window)
    assert (out[tokens:] == 0).all()
    at, want = 0, []
    for i, (n, held) in enumerate(segments):
        want.append(plain_fp4.attend(q[at:at + n].view(n, heads, dim), c.k[i], c.v[i], range(held, held + n), dim ** -0.5, window).view(n, -1))
        at += n
    close(out[:tokens], torch.cat(want), c.v, 2.0 ** -7)


def test_two_segments_of_one_request():
    heads, kv_heads, dim, page = 4, 2, 64, 16
    c = Filled([200], kv_heads, dim, page, seed=1)
    segments = [(0, 40, 20), (0, 1, 10), (0, 70, 130)]
    q = c.queries(111, heads, dim)
    ctx, group = step_of(segments, c.table.to(DEV), page)
    out = torch.empty(111, heads * dim, dtype=torch.bfloat16, device=DEV)
    attention(q.to(DEV), heads * dim, out, c.cache, group, ctx, heads, dim, 0.125)
    positions = [*range(20, 60), 10, *range(130, 200)]
    close(out, plain_fp4.attend(q.view(111, heads, dim), c.k[0], c.v[0], positions, 0.125).view(111, -1), c.v, 2.0 ** -7)


def test_captured_twice_and_replayed_at_once():
    """Two captured steps over the same cache, replayed on two streams at the same time with new inputs: neither touches the
    other's scratch."""
    heads, kv_heads, dim, page = 32, 8, 128, 16
    lengths = [400, 900, 77]
    c = Filled(lengths, kv_heads, dim, page, seed=6)
    graphs = []
    for i in range(2):
        ctx, group = step_of([(j, 1, n - 1 - 5 * i) for j, n in enumerate(lengths)], c.table.to(DEV), page)
        q = torch.zeros(3, heads * dim, dtype=torch.bfloat16, device=DEV)
        out = torch.zeros_like(q)
        run = lambda: attention(q, heads * dim, out, c.cache, group, ctx, heads, dim, dim ** -0.5)
        run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run()
        graphs.append((graph, q, out, ctx, group))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for turn in range(5):
        new = [c.queries(3, heads, dim) for _ in range(2)]
        for (_, q, _, _, _), x in zip(graphs, new):
            q.copy_(x.to(DEV))
        torch.cuda.synchronize()
        for (graph, *_), stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                for _ in range(20):
                    graph.replay()
        torch.cuda.synchronize()
        for i, ((_, _, out, _, _), x) in enumerate(zip(graphs, new)):
            want = torch.stack([plain_fp4.attend(x[j:j + 1].view(1, heads, dim), c.k[j], c.v[j], [n - 1 - 5 * i], dim ** -0.5).view(-1)
                                for j, n in enumerate(lengths)])
            close(out, want, c.v, 2.0 ** -10)


def test_same_bits_every_time():
    heads, kv_heads, dim, page = 32, 8, 128, 16
    lengths = [3000, 20, 1999, 640]
    c = Filled(lengths, kv_heads, dim, page, seed=8)
    ctx, group = step_of([(j, 1, n - 1) for j, n in enumerate(lengths)], c.table.to(DEV), page)
    q = c.queries(4, heads, dim).to(DEV)
    first = attention(q, heads * dim, torch.empty_like(q), c.cache, group, ctx, heads, dim, dim ** -0.5)
    for _ in range(20):
        assert torch.equal(first, attention(q, heads * dim, torch.empty_like(q), c.cache, group, ctx, heads, dim, dim ** -0.5))


def test_write_then_attend():
    """As a layer uses them: a prompt portion is written and attended to, then single tokens are."""
    heads, kv_heads, dim, page, eps = 8, 2, 128, 16, 1e-6
    table = torch.tensor([[4, 1, 7, 0, 2, 6]], dtype=torch.int32)
    cache = torch.zeros(ops().fp4_cache_shape(8, kv_heads, page, dim), dtype=torch.uint8, device=DEV)
    keys, values, done = [], [], 0
    for n in (70, 1, 1, 9, 1):
        qkv, (qw, kw), rot = inputs(n, heads, kv_heads, dim, dim, seed=done)
        positions = torch.arange(done, done + n)
        slots = table[0, positions // page] * page + positions % page
        x = qkv.double().view(n, heads + 2 * kv_heads, dim)
        keys.append(plain_fp4.held(rotated(normed(x[:, heads:heads + kv_heads], kw, eps), rot))[0])
        values.append(plain_fp4.held(x[:, heads + kv_heads:])[0])
        rows = qkv.to(DEV)
        ops().qk_norm_rope_cache_fp4(rows, heads, kv_heads, dim, to(qw), to(kw), eps, to(rot), dim, slots.int().to(DEV), cache)
        ctx, group = step_of([(0, n, done)], table.to(DEV), page)
        out = torch.empty(n, heads * dim, dtype=torch.bfloat16, device=DEV)
        attention(rows, rows.shape[1], out, cache, group, ctx, heads, dim, dim ** -0.5)
        q = rows[:, :heads * dim].cpu().view(n, heads, dim)        # the rounded queries: what the attention is given
        want = plain_fp4.attend(q, torch.cat(keys), torch.cat(values), positions.tolist(), dim ** -0.5).view(n, -1)
        close(out, want, values, 2.0 ** -7)
        done += n


@pytest.mark.parametrize("test", [
    test_calls_on_two_streams_at_once, test_many_tokens_of_a_launch_and_more, test_pages_that_are_not_held, test_large_and_small_magnitudes,
    test_nan_where_it_is_seen_and_only_there, test_captured_twice_and_replayed_at_once, test_same_bits_every_time, test_write_then_attend])
def test_the_same_dealt_to_all_blocks(monkeypatch, test):
    from mrun_b200.kernels import attention as module
    monkeypatch.setattr(module, "FP4_CLUSTER_TILES", (0, 0, 0))
    test()
