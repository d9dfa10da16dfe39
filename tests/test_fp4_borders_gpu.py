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
