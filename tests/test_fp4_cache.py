"""The 4-bit key/value cache without a device: its sizes in the cache manager's books, and what its entry points refuse."""
import pytest
import torch

import plain_fp4
from mrun_b200.kernels import KernelError, attention, ops


def test_a_unit_holds_every_value_once():
    for dim in (64, 128):
        places = [plain_fp4.code_at(dim, r, f, value) for value in (False, True) for r in range(16) for f in range(0, dim, 2)]
        places += [plain_fp4.scale_at(dim, r, s, value) for value in (False, True) for r in range(16) for s in range(dim // 16)]
        assert sorted(places) == list(range(ops.fp4_unit_bytes(dim)))


def test_what_groups_are_held_as():
    x = torch.zeros(16, dtype=torch.float64)
    x[:8] = torch.tensor([6.0, -6.0, 5.0, 2.5, -0.25, 0.75, 3.5, 0.3])
    values, code, byte = plain_fp4.held(x)
    assert values[:8].tolist() == [6.0, -6.0, 4.0, 2.0, 0.0, 1.0, 4.0, 0.5] and byte.item() == 120        # the scale is 1
    assert plain_fp4.held(1e9 * x)[0][:2].tolist() == [61440.0, -61440.0]
    assert plain_fp4.held(1e-9 * x)[0].abs().max() == 0
    x[3] = float("inf")
    assert torch.isnan(plain_fp4.held(x)[0]).all() and plain_fp4.held(x)[2].item() == 255
    assert torch.equal(plain_fp4.unit_of(torch.ones(16, 64), torch.ones(16, 64)), plain_fp4.units_of(torch.ones(16, 64), torch.ones(16, 64)))


def test_sizes_and_refusals():
    assert ops.fp4_unit_bytes(128) == 2304 and ops.fp4_unit_bytes(64) == 1152
    assert ops.fp4_cache_shape(5, 8, 48, 128) == (5, 8, 3, 2304)
    for bad in (0, 8, 24, -16):
        with pytest.raises(KernelError, match="multiple of 16"):
            ops.fp4_cache_shape(5, 8, bad, 128)
    for bad in (32, 96, 256):
        with pytest.raises(KernelError, match="64 or 128"):
            ops.fp4_unit_bytes(bad)


def _write(**change):
    args = dict(qkv=torch.zeros(3, 6 * 64, dtype=torch.bfloat16), heads=4, kv_heads=1, head_dim=64, q_weight=torch.ones(64),
                k_weight=torch.ones(64), eps=1e-6, rot=torch.zeros(3, 32, 2), rotary_dim=64, slots=torch.zeros(3, dtype=torch.int32),
                cache=torch.zeros(2, 1, 1, 1152, dtype=torch.uint8))
    args.update(change)
    return ops.qk_norm_rope_cache_fp4(**args)


@pytest.mark.parametrize("change, message", [
    (dict(heads=5), "expected width"), (dict(head_dim=32, heads=10, kv_heads=1), "64 or 128"),
    (dict(q_weight=torch.ones(32)), "q_weight has 32"), (dict(rot=torch.zeros(3, 16, 2)), "rot is"),
    (dict(slots=torch.zeros(2, dtype=torch.int32)), "one slot per token"), (dict(cache=None), "one slot per token"),
    (dict(cache=torch.zeros(2, 2, 1, 1152, dtype=torch.uint8)), "4-bit cache is"),
    (dict(cache=torch.zeros(2, 1, 1, 2304, dtype=torch.uint8)), "4-bit cache is"),
    (dict(q_out=torch.zeros(3, 64, dtype=torch.bfloat16)), "q_out is"),
    (dict(), "CUDA only"),
])
def test_write_refuses(change, message):
    with pytest.raises(KernelError, match=message):
        _write(**change)


def test_read_refuses():
    cache = torch.zeros(2, 1, 1, 1152, dtype=torch.uint8)
    with pytest.raises(KernelError, match="4-bit cache is"):
        ops.fp4_pages(cache, 128, torch.zeros(1, dtype=torch.int32))
    with pytest.raises(KernelError, match="expected a list"):
        ops.fp4_pages(cache, 64, torch.zeros(1, 1, dtype=torch.int32))
    with pytest.raises(KernelError, match="CUDA only"):
        ops.fp4_pages(cache, 64, torch.zeros(1, dtype=torch.int32))


class _Step:
    num_tokens = real_tokens = 3
    page_size = 16


def test_attention_refuses():
    cache = torch.zeros(2, 2, 1, 1152, dtype=torch.uint8)
    q, out = torch.zeros(3, 256, dtype=torch.bfloat16), torch.zeros(3, 256, dtype=torch.bfloat16)
    call = lambda q=q, stride=256, out=out, heads=4, dim=64: attention.paged_attention_fp4(q, stride, out, cache, None, _Step, heads, dim, 0.125)
    with pytest.raises(KernelError, match="not a multiple"):
        call(heads=5)
    with pytest.raises(KernelError, match="4-bit cache is"):
        call(dim=128)
    with pytest.raises(KernelError, match="out is"):
        call(heads=2)
    with pytest.raises(KernelError, match="strides"):
        call(stride=128)
    with pytest.raises(KernelError, match="strides"):
        call(q=torch.zeros(2, 256, dtype=torch.bfloat16))
    _Step.page_size = 32
    with pytest.raises(KernelError, match="pages of 16"):
        call()
    _Step.page_size = 16
    with pytest.raises(KernelError, match="CUDA only"):
        call()


def test_the_books_count_what_pages_take():
    from mrun_b200.cache import CacheManager, PagedKV, token_bytes
    from mrun_b200.cache.manager import read_back_bytes
    needs = [PagedKV(8, 128, fp4=True)] * 36
    assert token_bytes(needs, [None] * 36, 2) == (36 * 8 * 144, 0) == token_bytes(needs, [None] * 36, 4)
    assert token_bytes([PagedKV(4, 64, fp4=True), None, PagedKV(8, 128)], [None, 0, None], 2)[0] == 4 * 72 + 8 * 128 * 4
    assert read_back_bytes(needs) == 8 * 128 * 4 and read_back_bytes([PagedKV(8, 128), None]) == 0
    assert CacheManager(needs, [None] * 36, 16, 10, 2).bytes_per_page() == 0            # the books alone hold no pages
    with pytest.raises(ValueError, match="one size"):
        CacheManager([PagedKV(8, 128, value_dim=64, fp4=True)], [None], 16, 10, 2)


def test_a_budget_leaves_room_to_read_a_layer_back():
    from types import SimpleNamespace
    from mrun_b200.cache import PagedKV
    from mrun_b200.engine import budget
    from mrun_b200.engine.engine import _sizing
    from mrun_b200.engine.model import Model
    m = Model.__new__(Model)
    m.spec = SimpleNamespace(hidden_size=256, vocab_size=1000, max_positions=1 << 22)
    m.runtime = SimpleNamespace(precision=SimpleNamespace(act=torch.bfloat16))
    m.final_norm, m.embedding, m.head, m.embedder = None, torch.empty(8, 256), torch.empty(8, 256), None
    m.order, m.blocks = [], []
    m.cache_needs, m.cache_shares = (lambda: [PagedKV(8, 128, fp4=True)] * 4), (lambda: [None] * 4)
    memory = budget.plan(budget.DeviceMemory(80 * budget.GIB, 80 * budget.GIB), 4)
    pages, done = _sizing(memory, None, 16, 4, 512)(m)
    held, back = 4 * 8 * 144, 4 * 8 * 128
    fixed = done.scratch - done.capacity_tokens * back
    assert done.cache == done.capacity_tokens * held and pages == -(-done.capacity_tokens // 16)
    assert done.budget - held - back < done.weights + done.scratch + done.cache <= done.budget
    assert fixed == budget.scratch_estimate(256, 0, 1000, 512, 4, 2) + m.product_scratch(512)
    exactly = _sizing(memory, 5000, 16, 4, 512)(m)[1]
    assert exactly.capacity_tokens == 5000 and exactly.budget == exactly.weights + exactly.scratch + exactly.cache


def _spec(kind):
    from types import SimpleNamespace
    return SimpleNamespace(validate=lambda: None, streams=1, embedding_transform=None, layers=[SimpleNamespace(mixer=SimpleNamespace(kind=kind))])


def test_models_that_do_not_hold_their_cache_in_4_bits_are_refused():
    from mrun_b200.engine.model import Model
    from mrun_b200.parts import Precision, Runtime
    runtime = lambda kv_cache: Runtime(torch.device("cpu"), Precision.of("bfloat16"), 16, kv_cache)
    with pytest.raises(ValueError, match="layer 0: the mixer 'latent_attention' does not hold"):
        Model(_spec("latent_attention"), {}, runtime("fp4"))
    with pytest.raises(ValueError, match="kv_cache must be one of auto, fp4, got 'fp8'"):
        Model(_spec("attention"), {}, runtime("fp8"))


def test_an_attention_layer_refuses_what_the_format_does_not_hold():
    from mrun_b200.config.spec import AttentionSpec
    from mrun_b200.parts import MIXERS, Precision, Runtime
    spec = lambda dim: AttentionSpec(hidden=32, heads=4, kv_heads=2, head_dim=dim, softmax_scale=1.0, qk_norm=None, position=None)
    build = lambda dim, page, dtype: MIXERS.build(spec(dim), {}, Runtime(torch.device("cpu"), Precision.of(dtype), page, "fp4"))
    with pytest.raises(ValueError, match="bfloat16 activations"):
        build(64, 16, "float32")
    with pytest.raises(KernelError, match="multiple of 16"):
        build(64, 8, "bfloat16")
    with pytest.raises(KernelError, match="64 or 128"):
        build(96, 16, "bfloat16")
