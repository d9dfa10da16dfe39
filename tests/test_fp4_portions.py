"""What prompt portions over the 4-bit cache are planned as, without a device."""
import types

import pytest
import torch

from mrun_b200.engine.batch import SegmentInfo, StepContext
from mrun_b200.kernels import attention, ops


def step_of(segments, page=16):
    """A step over segments (slot, tokens, first position), on the host."""
    infos, at = [], 0
    for slot, n, first in segments:
        infos.append(SegmentInfo(slot, at, n, first))
        at += n
    positions = torch.cat([torch.arange(first, first + n, dtype=torch.int32) for _, n, first in segments])
    return StepContext(num_tokens=at, num_segments=len(infos), segments=infos, token_ids=None, positions=positions,
                       token_slot=torch.cat([torch.full((n,), slot, dtype=torch.int32) for slot, n, _ in segments]), seg_q_start=None,
                       seg_kv_len=None, seg_slot=None, groups={}, max_q_len=max(n for _, n, _ in segments),
                       max_kv_len=max(n + first for _, n, first in segments), page_size=page, real_tokens=at,
                       pages_held=True)


class Calls:
    """Stands in for the device: what the read back and the kernels behind it are asked for."""

    def __init__(self, monkeypatch):
        self.rows, self.spans, self.prompts, self.fail = [], [], [], 0
        monkeypatch.setattr(ops, "_check", lambda *a, **k: None)
        monkeypatch.setattr(ops, "_check_device", lambda *a, **k: None)
        monkeypatch.setattr(ops, "fp4_spans", self.read_back)
        monkeypatch.setattr(attention, "_fp4_tokens", lambda *a, **k: self.rows.append(a[-1]))
        monkeypatch.setattr(attention, "paged_attention", lambda q, stride, out, cache, view, ctx, *a: self.prompts.append((view, ctx)))

    def read_back(self, cache, head_dim, block_tables, spans, pages, rows, table=None, span_of_row=None):
        if self.fail:
            self.fail -= 1
            raise torch.OutOfMemoryError("no room to read back")
        self.spans.append((spans, pages, table, span_of_row))
        return None, None


def attend(ctx, heads=8, kv_heads=2, dim=64, page=16, pages=64, window=0):
    q = torch.zeros(ctx.num_tokens, heads * dim, dtype=torch.bfloat16)
    cache = torch.zeros(ops.fp4_cache_shape(pages, kv_heads, page, dim), dtype=torch.uint8)
    tables = torch.zeros(8, 64, dtype=torch.int32)
    group = types.SimpleNamespace(block_tables=tables)
    return attention.paged_attention_fp4(q, q.shape[1], torch.empty_like(q), cache, group, ctx, heads, dim, 0.125, window)


def test_a_call_that_failed_leaves_no_tables_that_nobody_wrote(monkeypatch):
    """The step's tables are memory as it comes until a read back has written them: a second call with the step must not take them
    for written because a first one began."""
    calls = Calls(monkeypatch)
    ctx = step_of([(0, 300, 0), (1, 200, 40)])
    calls.fail = 1
    with pytest.raises(torch.OutOfMemoryError):
        attend(ctx)
    for _ in range(2):
        attend(ctx)
    assert len(calls.spans) == len(calls.prompts) == 2
    for (spans, _, table, span_of_row), (view, inner) in zip(calls.spans, calls.prompts):
        assert table is not None and span_of_row is not None and len(spans) == 2
        assert view.block_tables.data_ptr() == table.data_ptr() and inner.token_slot.data_ptr() == span_of_row.data_ptr()
