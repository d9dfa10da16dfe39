"""The 4-bit cache where a rounding, a sign or the range of 32 bits decides: bytes against the definition, scores far from zero."""
import math

import pytest
import torch

import plain_fp4
from test_fp4_cache_gpu import DEV, Filled, attention, close, inputs, normed, ops, rotated, step_of, to

pytestmark = pytest.mark.gpu


def signs_and_borders(dim):
    """16 rows: zeros of either sign beside large and tiny values, borders between codes, groups that are zeros or infinite."""
    v = torch.zeros(16, dim)
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0])
    for i in range(dim // 8):
        v[0, 8 * i:8 * i + 8] = ties * 2.0 ** (i % 8 - 4) * (-1) ** i
    v[1] = -0.0
    v[2, ::2], v[2, 1::3] = -0.0, 6.0
    v[3, ::2], v[3, 1::2] = -1e-30, 3.0                        # round to zero and keep their sign
    v[4, ::2], v[4, 1::2] = -1e-30, 1e-30                      # a group whose scale is zero
    v[5, ::3], v[5, 1::3] = -0.0, -1e-38
    v[6, :16], v[6, 16:32], v[6, 32:48], v[6, 48:64] = 6 * 17 / 16, -6 * 19 / 16, 6 * 2.0 ** -18, -6 * 2.0 ** -17 * 1.5
    v[7, ::5] = -0.0
    v[7, 3], v[7, 20], v[7, 40] = math.inf, -math.inf, math.nan
    g = torch.Generator().manual_seed(3)
    v[8:] = torch.randn(8, dim, generator=g) * torch.exp(4 * torch.randn(8, dim, generator=g))
    v[8:, ::7] = -0.0
    return v.bfloat16()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("norm, rotary", [(False, 0), (True, 0), (False, 32), (True, 32), (True, 20)])
def test_bytes_of_zeros_and_borders(dim, norm, rotary):
    """Every byte of the page.  A zero of either sign is code 0; a value below zero has the sign bit, also where it rounds to zero."""
    v = signs_and_borders(dim)
    qkv = torch.cat([v, v, v], 1)
    g = torch.Generator().manual_seed(4)
    weight = (1 + 0.2 * torch.randn(dim, generator=g)) if norm else None
    rot = None
    if rotary:
        angle = torch.rand(16, rotary // 2, generator=g).double() * 6
        rot = torch.stack([angle.cos(), angle.sin()], -1).float()
    cache = torch.zeros(ops().fp4_cache_shape(1, 1, 16, dim), dtype=torch.uint8, device=DEV)
    ops().qk_norm_rope_cache_fp4(qkv.to(DEV), 1, 1, dim, to(weight), to(weight), 1e-6, to(rot), rotary, torch.arange(16, dtype=torch.int32, device=DEV),
                                 cache)
    k = rotated(normed(v.double().view(16, 1, dim), weight, float(torch.tensor(1e-6))), rot).view(16, dim)
    assert torch.equal(cache.view(-1).cpu(), plain_fp4.unit_of(k, v.double()))


@pytest.mark.parametrize("factor", [1.0, 1e3, 1e6])
@pytest.mark.parametrize("norm", [True, False])
def test_keys_under_a_rotary_table_of_any_size(factor, norm):
    """Pairs whose two products all but cancel, under tables of any size: the bound within which a key is computed in 32 bits follows the
    products, not the features alone."""
    dim, tokens, page = 128, 1500, 16
    qkv, (qw, kw), _ = inputs(tokens, 1, 1, dim, 0, seed=11, norm=norm)
    x = normed(qkv.double().view(tokens, 3, dim)[:, 1:2], kw, float(torch.tensor(1e-6)))
    g = torch.Generator().manual_seed(6)
    a, b = x[:, 0, :dim // 2], x[:, 0, dim // 2:]
    size = factor * torch.rand(tokens, dim // 2, generator=g).double() / torch.maximum(a.abs(), b.abs()).clamp(min=1e-3)
    rot = torch.stack([size * b, size * a * (1 + 1e-3 * torch.randn(tokens, dim // 2, generator=g).double())], -1).float()
    pages = -(-tokens // page)
    cache = torch.zeros(ops().fp4_cache_shape(pages, 1, page, dim), dtype=torch.uint8, device=DEV)
    ops().qk_norm_rope_cache_fp4(qkv.to(DEV), 1, 1, dim, to(qw), to(kw), 1e-6, to(rot), dim, torch.arange(tokens, dtype=torch.int32, device=DEV), cache)
    k = ops().fp4_pages(cache, dim, torch.arange(pages, dtype=torch.int32, device=DEV))[0]
    k = k.transpose(1, 2).reshape(-1, 1, dim)[:tokens].double().cpu()
    assert torch.equal(k, plain_fp4.held(rotated(x, rot))[0])


def rows_of(values, dim):
    return torch.tensor(values, dtype=torch.float64).view(-1, 1, 1).expand(-1, 1, dim).contiguous()


def fill(c, k, v):
    """Writes float64 keys and values [n, 1, dim] into the pages of request 0 (16 keys a page)."""
    units = -(-k.shape[0] // 16)
    pad = lambda x: torch.cat([x, torch.zeros(units * 16 - x.shape[0], *x.shape[1:], dtype=torch.float64)]).view(units, 16, 1, -1).transpose(1, 2)
    packed = plain_fp4.units_of(pad(k), pad(v))
    for b in range(units):
        c.cache[int(c.table[0, b]), :, 0] = packed[b].to(DEV)


@pytest.mark.parametrize("tiles", [None, 0])
@pytest.mark.parametrize("heads, n", [(1, 1), (4, 40), (8, 700)])
def test_scores_near_the_end_of_32_bits(monkeypatch, tiles, heads, n):
    """Every score of a row below -1e38: the row still is the softmax of them (here the value of the least negative one)."""
    from mrun_b200.kernels import attention as module
    if tiles is not None:
        monkeypatch.setattr(module, "FP4_CLUSTER_TILES", (tiles,) * 3)
    dim = 64
    c = Filled([n], 1, dim, 16, seed=1)
    g = torch.Generator().manual_seed(n)
    size = torch.tensor([61440.0, 43008.0])[torch.randint(0, 2, (n,), generator=g)]
    size[n // 2] = 6 * 5120.0
    k, v = rows_of(size.tolist(), dim), torch.randn(n, 1, dim, generator=g).double()
    fill(c, k, v)
    k, v = plain_fp4.held(k)[0], plain_fp4.held(v)[0]
    assert torch.equal(k[:, 0, 0].float(), size)
    for sign in (-1.0, 1.0):
        q = torch.full((1, heads * dim), sign * 2.0 ** 105).bfloat16()
        size[n // 2] = 6 * 5120.0 if sign < 0 else 61440.0
        score = q[0, 0].double() * dim * k[:, 0, 0] * 1.4426950408889634
        assert score.abs().min() > 1e38 and score.abs().max() < 3e38
        if sign > 0 and n > 1:          # one key above the others
            size = torch.full((n,), 43008.0)
            size[n // 3] = 61440.0
            k = rows_of(size.tolist(), dim)
            fill(c, k, v)
        ctx, group = step_of([(0, 1, n - 1)], c.table.to(DEV), 16)
        out = torch.empty(1, heads * dim, dtype=torch.bfloat16, device=DEV)
        attention(q.to(DEV), heads * dim, out, c.cache, group, ctx, heads, dim, 1.0)
        close(out, plain_fp4.attend(q.view(1, heads, dim), k, v, [n - 1], 1.0).view(1, -1), [v], 2.0 ** -10)


@pytest.mark.parametrize("tiles", [None, 0])
def test_keys_of_zeros_under_a_scale_that_leaves_the_range(monkeypatch, tiles):
    """2^126 times 2^10 is no 32-bit number, its product with a key of zeros is 0: the mean of the values."""
    from mrun_b200.kernels import attention as module
    if tiles is not None:
        monkeypatch.setattr(module, "FP4_CLUSTER_TILES", (tiles,) * 3)
    heads, dim, n = 4, 128, 50
    c = Filled([n], 1, dim, 16, seed=1)
    v = torch.randn(n, 1, dim, generator=torch.Generator().manual_seed(2)).double()
    fill(c, torch.zeros_like(v), v)
    v = plain_fp4.held(v)[0]
    q = torch.full((1, heads * dim), 2.0 ** 126).bfloat16()
    ctx, group = step_of([(0, 1, n - 1)], c.table.to(DEV), 16)
    out = torch.empty(1, heads * dim, dtype=torch.bfloat16, device=DEV)
    attention(q.to(DEV), heads * dim, out, c.cache, group, ctx, heads, dim, 2.0 ** 10)
    close(out, v.mean(0).repeat(1, heads).view(1, -1), [v], 2.0 ** -10)


def test_rows_for_q_that_lie_in_the_projection_are_refused():
    """Other lanes still read the keys, the values or other rows there.  The projection's own q columns are written in place."""
    from mrun_b200.kernels import KernelError
    heads, kv_heads, dim, tokens = 2, 2, 64, 5
    qkv, (qw, kw), rot = inputs(tokens, heads, kv_heads, dim, dim, seed=1)
    memory = torch.zeros(3 * tokens, 3 * heads * dim, dtype=torch.bfloat16, device=DEV)
    rows, wide = memory[tokens:2 * tokens], heads * dim
    rows.copy_(qkv)
    cache = torch.zeros(ops().fp4_cache_shape(1, kv_heads, 16, dim), dtype=torch.uint8, device=DEV)
    slots = torch.arange(tokens, dtype=torch.int32, device=DEV)
    call = lambda q_out: ops().qk_norm_rope_cache_fp4(rows, heads, kv_heads, dim, to(qw), to(kw), 1e-6, to(rot), dim, slots, cache, q_out=q_out)
    flat = memory.view(-1)
    for q_out in (rows[:, wide:2 * wide], rows[:, 2 * wide:], rows[:, 8:8 + wide], memory[tokens - 1:2 * tokens - 1, :wide],
                  memory[2 * tokens - 1:3 * tokens - 1, :wide], flat[tokens * 3 * wide:tokens * 4 * wide].view(tokens, wide)):
        with pytest.raises(KernelError, match="q_out lies in"):
            call(q_out)
    assert torch.equal(rows.cpu(), qkv) and not cache.any()
    apart = [call(memory[:tokens, :wide]).clone(), call(memory[2 * tokens:, wide:2 * wide]).clone()]
    assert torch.equal(rows.cpu(), qkv)
    assert torch.equal(call(rows[:, :wide]), apart[0]) and torch.equal(*apart)
