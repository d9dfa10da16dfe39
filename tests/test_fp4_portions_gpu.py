"""Prompt portions over the 4-bit cache: what their keys and values being read back must not change.  Tolerances are those of
``test_fp4_cache_gpu``: portions whose contexts are read back round P to bfloat16."""
import pytest
import torch

import plain_fp4
from test_fp4_cache_gpu import DEV, Filled, attention, close, step_of

pytestmark = pytest.mark.gpu


def wanted(c, q, segments, heads, dim, window, seen=None):
    """Float64 rows of the step; ``seen``: per segment, the keys whose page is held, or None."""
    at, out = 0, []
    for i, (slot, n, first) in enumerate(segments):
        if not 0 <= slot < len(c.k):
            out.append(torch.zeros(n, heads * dim, dtype=torch.float64))
        else:
            k, v = c.k[slot], c.v[slot]
            behind = max(0, first + n - k.shape[0])            # positions behind the table: keys that nobody sees
            mask = torch.ones(k.shape[0], dtype=torch.bool) if not seen or seen[i] is None else seen[i]
            mask = torch.cat([mask, torch.zeros(behind, dtype=torch.bool)])
            k, v = (torch.cat([x, x.new_zeros(behind, *x.shape[1:])]) for x in (k, v))
            out.append(plain_fp4.attend(q[at:at + n].view(n, heads, dim), k, v, range(first, first + n), dim ** -0.5, window, mask).view(n, -1))
        at += n
    return torch.cat(out)


@pytest.mark.parametrize("heads, kv_heads, dim, page, window", [
    (8, 2, 128, 16, 0), (8, 2, 64, 48, 0), (12, 3, 128, 64, 0), (6, 2, 64, 16, 100), (8, 2, 128, 16, -128), (2, 2, 64, 64, 150)])
def test_pages_that_are_not_held_in_long_portions(heads, kv_heads, dim, page, window):
    """Freed pages, page numbers outside the cache, tables without any page, requests outside the tables, positions behind the table: in
    segments of so many tokens that their keys are read back, beside segments whose pages are all held."""
    from mrun_b200.kernels import attention as module
    length = 576
    c = Filled([length] * 5, kv_heads, dim, page, seed=page + heads)
    table = c.table.clone()
    table[0, 64 // page], table[0, 384 // page], table[0, 448 // page] = -1, 10 ** 6, -1        # behind it, among its own tokens, twice
    table[2] = -1
    held = [torch.ones(length, dtype=torch.bool) for _ in range(5)]
    for key in (64, 384, 448):
        held[0][key // page * page:(key // page + 1) * page] = False
    held[2][:] = False
    segments = [(0, 300, 260), (1, 200, 33), (2, 150, 20), (9, 140, 0), (-4, 131, 400), (3, 310, length - 150), (4, 1, 500), (4, 160, 300)]
    seen = [held[s] if 0 <= s < 5 else None for s, _, _ in segments]
    tokens = sum(n for _, n, _ in segments)
    q = c.queries(tokens + 2, heads, dim)
    ctx, group = step_of(segments, table.to(DEV), page, tokens=tokens + 2)
    out = torch.full((tokens + 2, heads * dim), 3.0, dtype=torch.bfloat16, device=DEV)
    attention(q.to(DEV), heads * dim, out, c.cache, group, ctx, heads, dim, dim ** -0.5, window)
    assert len(module._fp4_portions(ctx, window, heads, kv_heads)[1][0]) == 7            # all but the single token
    assert (out[tokens:] == 0).all() and (out[500:650] == 0).all() and (out[650:921] == 0).all()
    close(out[:tokens], wanted(c, q, segments, heads, dim, window, seen), c.v, 2.0 ** -7)


def test_many_portions_with_pages_that_are_not_held():
    """More portions than a launch takes, every third with a hole."""
    heads, kv_heads, dim, page, n = 4, 1, 64, 16, 70
    c = Filled([160] * 70, kv_heads, dim, page, seed=5)
    table = c.table.clone()
    table[::3, 4] = -1
    hole = torch.ones(160, dtype=torch.bool)
    hole[64:80] = False
    segments = [(i, n + i % 3, 160 - n - i % 3) for i in range(70)]
    tokens = sum(s[1] for s in segments)
    q = c.queries(tokens, heads, dim)
    ctx, group = step_of(segments, table.to(DEV), page)
    out = torch.empty(tokens, heads * dim, dtype=torch.bfloat16, device=DEV)
    attention(q.to(DEV), heads * dim, out, c.cache, group, ctx, heads, dim, dim ** -0.5)
    close(out, wanted(c, q, segments, heads, dim, 0, [hole if i % 3 == 0 else None for i in range(70)]), c.v, 2.0 ** -7)


def test_a_step_whose_pages_are_held_is_not_looked_through():
    """The same bits with and without the look, which an engine's steps do not pay for."""
    from mrun_b200.kernels import lib
    heads, kv_heads, dim, page = 8, 2, 128, 16
    c = Filled([400], kv_heads, dim, page, seed=1)
    q = c.queries(300, heads, dim).to(DEV)
    outs, calls = [], []
    for held in (False, True):
        ctx, group = step_of([(0, 300, 100)], c.table.to(DEV), page)
        ctx.pages_held = held
        outs.append(torch.empty(300, heads * dim, dtype=torch.bfloat16, device=DEV))
        before = lib.call_count()
        attention(q, heads * dim, outs[-1], c.cache, group, ctx, heads, dim, dim ** -0.5)
        calls.append(lib.call_count() - before)
    assert torch.equal(*outs) and calls[0] == calls[1] + 1


def test_spans_that_leave_pages_or_name_no_row_are_refused():
    """Pages that no span takes would come back as memory that nobody wrote; a row number of more than 32 bits is not cut to another row."""
    from mrun_b200.kernels import KernelError, ops
    c = Filled([100], 2, 64, 16)
    table = c.table.to(DEV)
    for spans, pages, rows in (([(0, 0, 100, 0, 0, 4)], 3, 64), ([], 1, 64), ([(0, 0, 64, 0, 0, 4)], 2, 64), ([(1 << 32, 0, 100, 0, 0, 4)], 2, 64),
                               ([(-1 << 33, 0, 100, 0, 0, 4)], 2, 64), ([(0, 0, 100, 0, 0, 4)], 2, 0), ([(0, 0, 100, 0, 0, 4)], 2, 60)):
        with pytest.raises(KernelError):
            ops.fp4_spans(c.cache, 64, table, spans, pages, rows)
    k, v = ops.fp4_spans(c.cache, 64, table, [(0, 0, 64, 0, 0, 1), (-7, 0, 65, 1, 0, 1), (0, 64, 100, 3, 0, 1)], 4, 64)
    got = torch.cat([k[0], k[3]], 1).double().cpu().transpose(0, 1)
    assert torch.equal(got[:100], c.k[0]) and not got[100:].any() and not k[1:3].any() and not v[1:3].any()
    assert [x.shape[0] for x in ops.fp4_spans(c.cache, 64, table, [], 0, 64)] == [0, 0]


@pytest.mark.parametrize("heads, kv_heads, dim, page, lengths, window", [
    (8, 2, 128, 16, [150, 170, 300, 33], 0), (12, 3, 64, 48, [130, 300, 97], 0), (8, 2, 128, 64, [129, 200], 0), (8, 2, 64, 256, [300, 290], 0),
    (8, 2, 128, 32, [400, 390], 100), (4, 2, 64, 16, [400, 390], -128)])
def test_a_cache_that_is_full(heads, kv_heads, dim, page, lengths, window):
    """No page is free: what is read back takes the cache's own pages in place of ones of 128 rows.  The bits are those of a cache with room."""
    from mrun_b200.kernels import attention as module
    c = Filled(lengths, kv_heads, dim, page, seed=7, spare=40)
    segments = [(i, n - n // 4, n // 4) for i, n in enumerate(lengths)]
    table = c.table.clone()
    for i, (_, _, first) in enumerate(segments):               # what a window has passed is given back
        table[i, :plain_fp4.first_visible(first, window) // page] = -1
    kept = table[table >= 0].long()
    new = torch.full((c.cache.shape[0],), -1, dtype=torch.int32)
    new[kept] = torch.arange(kept.numel(), dtype=torch.int32)
    full_table = torch.where(table >= 0, new[table.clamp(min=0).long()], table)
    q = c.queries(sum(n for _, n, _ in segments), heads, dim)
    outs, sizes = [], []
    for cache, block_table in ((c.cache, table), (c.cache[kept.to(DEV)].contiguous(), full_table)):
        ctx, group = step_of(segments, block_table.to(DEV), page)
        outs.append(torch.empty(q.shape, dtype=torch.bfloat16, device=DEV))
        attention(q.to(DEV), heads * dim, outs[-1], cache, group, ctx, heads, dim, dim ** -0.5, window)
        close(outs[-1], wanted(c, q, segments, heads, dim, window), c.v, 2.0 ** -7)
        longer = module._fp4_portions(ctx, window, heads, kv_heads, cache.shape[0] * page)[1]
        sizes.append(longer[4].page_size)
        assert longer[1] * sizes[-1] <= cache.shape[0] * page
    assert sizes[0] == 128 and torch.equal(*outs)
