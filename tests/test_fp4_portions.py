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


def portioned(segments, heads=32, kv_heads=8, window=0):
    """(rows that go one by one, slots of the segments that are read back)."""
    rows, longer = attention._fp4_portions(step_of(segments), window, heads, kv_heads)
    return rows, [] if longer is None else sorted(span[0] for span in longer[0])


def rows_of(segments, slots):
    at, out = 0, []
    for slot, n, _ in segments:
        out += range(at, at + n) if slot in slots else []
        at += n
    return out


@pytest.mark.parametrize("decoding", [8, 33, 64, 300])
@pytest.mark.parametrize("n", [4, 16, 30, 32])
def test_decoding_tokens_leave_short_portions_their_way(decoding, n):
    """A few tokens behind a context go by rows whatever the number of decoding requests beside them."""
    segments = [(i, 1, 2000 + i) for i in range(decoding)] + [(decoding, n, 2100)]
    rows, back = portioned(segments)
    assert not back and sorted(rows) == list(range(decoding + n))


@pytest.mark.parametrize("heads, kv_heads, count, n, by_rows", [
    (32, 8, 1, 32, True), (32, 8, 2, 32, False), (32, 8, 8, 32, False), (32, 8, 16, 16, True), (32, 8, 17, 16, False), (32, 8, 24, 16, False),
    (16, 16, 4, 32, True), (16, 16, 5, 32, False), (16, 16, 8, 32, False), (128, 1, 3, 200, True)])
def test_segments_of_a_kind_go_the_same_way(heads, kv_heads, count, n, by_rows):
    segments = [(i, n, 9000) for i in range(count)]
    rows, back = portioned(segments, heads, kv_heads)
    assert (sorted(rows), back) == ((list(range(count * n)), []) if by_rows else ([], list(range(count))))


def test_the_two_kinds_are_decided_apart():
    segments = [(0, 16, 9000), (1, 1500, 0), (2, 1, 50), (3, 30, 2100), (4, 5, 0)]
    rows, back = portioned(segments)
    assert back == [1, 3] and sorted(rows) == rows_of(segments, (0, 2, 4))
    segments = [(i, 16, 100) for i in range(17)] + [(17, 20, 100)]
    rows, back = portioned(segments)
    assert back == list(range(17)) and sorted(rows) == rows_of(segments, (17,))


@pytest.mark.parametrize("page, lengths, window", [
    (16, [33] * 64, 0), (16, [150, 17, 300, 1000], 0), (48, [50] * 9, 0), (64, [65, 70, 200], 0), (256, [300, 257, 900], 0), (32, [700, 650, 800], 100),
    (16, [700] * 5, -256), (16, [2000], 0)])
def test_what_is_read_back_is_no_more_than_the_cache(monkeypatch, page, lengths, window):
    """A memory budget sets aside the read back of as many tokens as the cache holds: also where the cache is full of short requests, each of
    which would be rounded up to 128 tokens."""
    calls = Calls(monkeypatch)
    held = [(0 if window == 0 else attention._first_visible(n - n // 2, window) // page, -(-n // page)) for n in lengths]
    pool = sum(end - first for first, end in held)
    for pages in (pool, 20 * pool + 40):
        ctx = step_of([(i, n // 2, n - n // 2) for i, n in enumerate(lengths)], page)
        monkeypatch.setattr(attention, "FP4_ROWS", 0)
        monkeypatch.setattr(attention, "FP4_ROWS_OF_A_TILE", 0)
        attend(ctx, page=page, pages=pages, window=window)
        spans, taken, table, _ = calls.spans[-1]
        inner = calls.prompts[-1][1]
        assert taken * inner.page_size <= pages * page and 128 % inner.page_size == 0 and inner.page_size >= 16
        at = 0
        for (slot, first, end, page0, _, _), n in zip(sorted(spans, key=lambda span: span[3]), sorted(lengths)):
            assert page0 == at and end == n and first % inner.page_size == 0 and first <= attention._first_visible(n - n // 2, window)
            at += -(-(end - first) // inner.page_size)
            assert -(-end // inner.page_size) <= table.shape[1]
        assert at == taken
    assert inner.page_size == 128


def test_a_step_is_described_as_before():
    """Callers that give a step's fields in their order still do; a step that says nothing of its pages has them looked through."""
    from dataclasses import fields
    assert [f.name for f in fields(StepContext)][-4:] == ["real_tokens", "upload", "shared", "pages_held"]
    assert next(f.default for f in fields(StepContext) if f.name == "pages_held") is False


@pytest.mark.parametrize("segments", [[(0, 1, 5)], [(0, 300, 0)], [(0, 300, 0), (1, 1, 9)]])
@pytest.mark.parametrize("scale", [0.0, -0.125, float("nan"), float("inf")])
def test_a_scale_that_is_not_positive_is_refused_before_anything_runs(monkeypatch, segments, scale):
    calls = Calls(monkeypatch)
    q = torch.zeros(sum(n for _, n, _ in segments), 512, dtype=torch.bfloat16)
    cache = torch.zeros(ops.fp4_cache_shape(4, 2, 16, 64), dtype=torch.uint8)
    with pytest.raises(ops.KernelError, match="scale"):
        attention.paged_attention_fp4(q, 512, torch.empty_like(q), cache, types.SimpleNamespace(block_tables=torch.zeros(8, 64, dtype=torch.int32)),
                                      step_of(segments), 8, 64, scale)
    assert not calls.rows and not calls.spans and not calls.prompts
