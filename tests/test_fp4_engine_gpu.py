"""A model whose keys and values are held in 4 bits: the attention layer, whole models under several cuttings, captured
decoding, and the command line."""
from __future__ import annotations

import json
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import plain_fp4
import plain_qwen3 as plain
from tiny_models import TINY, TOLERANCE, make_folder, random_tokens, rel_error, tiny_config

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
ROOT = os.path.normpath(os.path.join(os.path.dirname(os.path.abspath(__file__)), os.pardir))
NAMES = ("C", "E")           # the tiny models with heads of 64 and of 128


def held_block(h, w, prefix, cfg, positions, window=None):
    """``plain.attention_block`` with the keys and values as a 4-bit cache holds them."""
    nh, nkv, D = cfg["num_attention_heads"], cfg["num_key_value_heads"], plain.head_dim_of(cfg)
    q, k, v = ((h @ w[f"{prefix}.{n}_proj.weight"].T).view(h.shape[0], -1, D) for n in "qkv")
    q, k = (plain.rms_norm(x, w[f"{prefix}.{n}_norm.weight"], cfg["rms_norm_eps"]) for x, n in ((q, "q"), (k, "k")))
    q, k = (plain.rope(x, positions, plain.rope_theta_of(cfg)) for x in (q, k))
    k, v = (plain_fp4.held(x)[0].float() for x in (k, v))
    o = plain.attention_scores_softmax_values(q, k, v, float(D) ** -0.5, positions, window)
    return o.reshape(h.shape[0], nh * D) @ w[f"{prefix}.o_proj.weight"].T


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("chunks", [[50], [5, 2, 30, 1, 12], [1] * 20, [130, 1, 3, 80]])
def test_attention_part(name, chunks):
    """The layer against 64 bits from the products it makes itself: norms, rotation, held keys and values, attention, output."""
    from mrun_b200.cache import CacheManager
    from mrun_b200.engine.batch import HostStaging, StepEntry, build_context
    from mrun_b200.kernels import ops
    from mrun_b200.parts import MIXERS, Precision, Runtime
    from mrun_b200.weights import random_tensors
    config = tiny_config(name)
    spec = config.to_spec().layers[0].mixer
    tensors = dict(random_tensors(config.to_spec(), 1, std=TINY[name]["std"], norm_noise=0.1, dtype=torch.bfloat16))
    local = {k.split("layers.0.self_attn.")[1]: v for k, v in tensors.items() if "layers.0.self_attn." in k}
    rt = Runtime(torch.device(DEV), Precision.of("bfloat16"), 16, "fp4")
    part = MIXERS.build(spec, local, rt)
    manager = CacheManager([part.cache_need()], [None], 16, 64, 2, device=rt.device, dtype=rt.precision.act)
    assert manager.entries[0].k is None and manager.bytes_per_page() == 16 * spec.kv_heads * (spec.head_dim + spec.head_dim // 8)
    request, staging = manager.admit("r"), HostStaging(rt.device)
    g = torch.Generator().manual_seed(3)
    keys, values, start = [], [], 0
    H, G, D = spec.heads, spec.kv_heads, spec.head_dim
    for n in chunks:
        x = torch.randn(n, config.hidden_size, generator=g).bfloat16().to(DEV)
        plan = manager.plan_append([(request, n)])
        ctx = build_context([StepEntry(request, [1] * n)], manager, staging)
        got = part.forward(x, ctx, manager.entries[0]).double().cpu()
        manager.commit(plan)
        qkv = ops.linear(x, part.wqkv).cpu().float().view(n, H + 2 * G, D)
        positions = torch.arange(start, start + n)
        q, k = (plain.rope(plain.rms_norm(y.double(), local[f"{w}_norm.weight"].double(), spec.qk_norm.eps), positions, config.rope_theta)
                for y, w in ((qkv[:, :H], "q"), (qkv[:, H:H + G], "k")))
        keys.append(plain_fp4.held(k)[0]); values.append(plain_fp4.held(qkv[:, H + G:].double())[0])
        want = plain_fp4.attend(q, torch.cat(keys), torch.cat(values), positions.tolist(), spec.softmax_scale).view(n, H * D)
        want = want @ local["o_proj.weight"].double().T
        # q, P, the heads' output and the product's rows are each rounded to 16 bits: 3e-2 of the largest, as for the 16-bit cache
        assert (got - want).abs().max() <= 3e-2 * want.abs().max()
        start += n


@pytest.mark.parametrize("name", NAMES)
def test_logits_under_every_cutting(name, tmp_path, monkeypatch):
    """Whole prompts, portions, token by token through captured steps: the logits of the plain model with held keys and values.
    Rounding to bfloat16 in front of a key or value moves some of them over a border between two codes; each moves by at most a step,
    as holding them in 4 bits moved them, so the bound is the one of the 16-bit cache plus what holding changes."""
    from mrun_b200.engine import StepEntry
    from mrun_b200.engine.loading import executor_from_folder
    folder = make_folder(name, str(tmp_path / "m"))
    cfg, weights = plain.load_folder(folder)
    tokens = random_tokens(cfg["vocab_size"], 200, seed=5)
    exact = plain.forward(cfg, weights, tokens).numpy()
    monkeypatch.setattr(plain, "attention_block", held_block)
    want = plain.forward(cfg, weights, tokens).numpy()
    allowed = TOLERANCE["bfloat16"] + rel_error(exact, want)
    ex = executor_from_folder(folder, num_pages=64, max_requests=4, kv_cache="fp4")
    for sizes in ([200], [70, 3, 1, 126], [1] * 40 + [160]):
        request, at, got = ex.admit("r"), 0, []
        for n in sizes:
            got.append(ex.step([StepEntry(request, tokens[at:at + n], range(n))]).cpu().numpy())
            at += n
        assert rel_error(np.concatenate(got), want) <= allowed
        ex.release(request)
    first, second = ex.admit("a"), ex.admit("b")
    ex.step([StepEntry(first, tokens[:30], [])])
    ex.step([StepEntry(second, tokens[:77], [])])
    for i in range(60):
        ex.decode_step([StepEntry(first, [tokens[30 + i]], [0]), StepEntry(second, [tokens[77 + i]], [0])])
        got = ex.decode_logits([None, None]).cpu().numpy()
        assert rel_error(got, want[[30 + i, 77 + i]]) <= allowed
    # a prompt portion beside a decoding request
    mixed = ex.step([StepEntry(first, [tokens[90]], [0]), StepEntry(second, tokens[137:190], [52])]).cpu().numpy()
    assert rel_error(mixed, want[[90, 189]]) <= allowed
    ex.trim(first, 40)
    again = ex.step([StepEntry(first, tokens[40:50], range(10))]).cpu().numpy()
    assert rel_error(again, want[40:50]) <= allowed
    ex.check()
    ex.cache.check_invariants()


def test_captured_steps_of_several_bounds(tmp_path, monkeypatch):
    """A request that grows past the bounds of its captured steps, beside a short one: the logits of the plain model."""
    from mrun_b200.engine import StepEntry
    from mrun_b200.engine.loading import executor_from_folder
    folder = make_folder("E", str(tmp_path / "m"))
    cfg, weights = plain.load_folder(folder)
    tokens = random_tokens(cfg["vocab_size"], 150, seed=6)
    exact = plain.forward(cfg, weights, tokens).numpy()
    monkeypatch.setattr(plain, "attention_block", held_block)
    want = plain.forward(cfg, weights, tokens).numpy()
    allowed = TOLERANCE["bfloat16"] + rel_error(exact, want)
    assert executor_from_folder(folder, num_pages=8, max_requests=2).REACHES == (4096, 16384)
    ex = executor_from_folder(folder, num_pages=32, max_requests=2, kv_cache="fp4")
    assert ex.REACHES == (2048, 4096, 16384)
    ex.REACHES = (40, 100)
    long, short = ex.admit("long"), ex.admit("short")
    ex.step([StepEntry(long, tokens[:30], [])])
    ex.step([StepEntry(short, tokens[:2], [])])
    for i in range(110):
        ex.decode_step([StepEntry(long, [tokens[30 + i]], [0]), StepEntry(short, [tokens[2 + i]], [0])])
        got = ex.decode_logits([None, None]).cpu().numpy()
        assert rel_error(got, want[[30 + i, 2 + i]]) <= allowed
    assert [reach for reach in ex._graphs[2] if reach <= 100] == [40, 100] and len(ex._graphs[2]) == 3


def test_generation_is_the_same_every_time_and_in_company(tmp_path):
    from mrun_b200 import Engine
    folder = make_folder("E", str(tmp_path / "m"))
    prompts = [random_tokens(TINY["E"]["config"]["vocab_size"], n, seed=n) for n in (1, 9, 40, 171)]
    engine = Engine.from_folder(folder, context=1024, max_batch_tokens=64, max_requests=4, kv_cache="fp4")
    first = [r.tokens for r in engine.generate(prompts, max_tokens=30, ignore_eos=True)]
    assert engine.executor._graphs and all(len(t) == 30 for t in first)
    assert [r.tokens for r in engine.generate(prompts, max_tokens=30, ignore_eos=True)] == first
    info = engine.info()
    heads, dim = TINY["E"]["config"]["num_key_value_heads"], TINY["E"]["config"]["head_dim"]
    assert info["kv_cache"] == "fp4" and info["cache_bytes"] == info["capacity_tokens"] * 2 * heads * (dim + dim // 8)
    engine.executor.cache.check_invariants()


def test_command_line(tmp_path):
    from mrun_b200 import Engine
    folder = make_folder("C", str(tmp_path / "m"))
    prompt = random_tokens(300, 20, seed=1)
    run = lambda *args: subprocess.run([sys.executable, os.path.join(ROOT, "bin", "mrun"), "run", folder, *args], capture_output=True, text=True, timeout=600)
    result = run("--prompt", ",".join(map(str, prompt)), "--max-tokens", "8", "--ignore-eos", "--context", "1K", "--kv-cache", "fp4")
    assert result.returncode == 0, result.stderr
    engine = Engine.from_folder(folder, context=1024, max_requests=1, kv_cache="fp4")
    assert [int(t) for t in result.stdout.strip().split(",")] == engine.generate([prompt], max_tokens=8, ignore_eos=True)[0].tokens
    shown = run("--info", "--context", "1K", "--kv-cache", "fp4")
    info = json.loads(shown.stdout)
    assert info["kv_cache"] == "fp4" and info["memory"]["cache_bytes"] == 1024 * 2 * 2 * 72
    refused = run("--prompt", "1,2", "--kv-cache", "fp4", "--dtype", "float32")
    assert refused.returncode == 1 and "bfloat16 activations" in refused.stderr
