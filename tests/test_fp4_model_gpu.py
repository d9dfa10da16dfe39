"""Whole models with a 4-bit cache: that the held keys and values are what is attended to, in prompts and in captured steps, and that a
request's logits are its own whatever runs beside it."""
import numpy as np
import pytest

import plain_qwen3 as plain
from test_fp4_engine_gpu import held_block
from tiny_models import TOLERANCE, make_folder, random_tokens, rel_error

pytestmark = pytest.mark.gpu


def root_mean_square(a, b):
    return float(np.sqrt(np.mean((np.asarray(a, np.float64) - np.asarray(b, np.float64)) ** 2)))


def both(name, tmp_path, monkeypatch, tokens):
    """(folder, logits with the keys and values as they are, logits with them as a 4-bit cache holds them)."""
    folder = make_folder(name, str(tmp_path / "m"))
    cfg, weights = plain.load_folder(folder)
    tokens = random_tokens(cfg["vocab_size"], tokens, seed=12)
    exact = plain.forward(cfg, weights, tokens).numpy()
    monkeypatch.setattr(plain, "attention_block", held_block)
    return folder, tokens, exact, plain.forward(cfg, weights, tokens).numpy()


@pytest.mark.parametrize("name", ["C", "E"])
def test_logits_are_those_of_held_keys_and_values(name, tmp_path, monkeypatch):
    """Nearer to the model with held keys and values than to the one without, which an engine that kept 16 bits would not be; and the
    other way round without ``kv_cache``."""
    from mrun_b200.engine import StepEntry
    from mrun_b200.engine.loading import executor_from_folder
    folder, tokens, exact, held = both(name, tmp_path, monkeypatch, 200)
    for kv_cache, near, far in (("fp4", held, exact), ("auto", exact, held)):
        ex = executor_from_folder(folder, num_pages=64, max_requests=4, kv_cache=kv_cache)
        for sizes in ([200], [70, 3, 1, 126]):
            request, at, got = ex.admit("r"), 0, []
            for n in sizes:
                got.append(ex.step([StepEntry(request, tokens[at:at + n], range(n))]).cpu().numpy())
                at += n
            got = np.concatenate(got)
            assert root_mean_square(got, near) < root_mean_square(got, far)
            ex.release(request)
        request, got = ex.admit("captured"), []
        ex.step([StepEntry(request, tokens[:60], [])])
        for i in range(60, 200):
            ex.decode_step([StepEntry(request, [tokens[i]], [0])])
            got.append(ex.decode_logits([None]).cpu().numpy())
        assert ex._graphs
        got = np.concatenate(got)
        assert root_mean_square(got, near[60:]) < root_mean_square(got, far[60:])


def test_a_request_alone_and_in_company(tmp_path, monkeypatch):
    """Alone, beside decoding requests, and beside other prompts: within what the 16-bit cache's rounding and the borders between codes allow of
    the same logits."""
    from mrun_b200.engine import StepEntry
    from mrun_b200.engine.loading import executor_from_folder
    folder, tokens, exact, held = both("E", tmp_path, monkeypatch, 120)
    allowed = TOLERANCE["bfloat16"] + rel_error(exact, held)
    ex = executor_from_folder(folder, num_pages=128, max_requests=8, kv_cache="fp4")
    others = [ex.admit(f"other {i}") for i in range(4)]
    for i, other in enumerate(others):
        ex.step([StepEntry(other, tokens[i:i + 30 + 9 * i], [])])
    runs = {}
    for name in ("alone", "beside decoding", "beside prompts"):
        request, got = ex.admit(name), []
        for first, n in ((0, 90), (90, 4), (94, 1), (95, 25)):
            entries = [StepEntry(request, tokens[first:first + n], range(n))]
            if name == "beside decoding":
                entries += [StepEntry(other, [tokens[first % 50]], []) for other in others]
            elif name == "beside prompts":
                entries = [StepEntry(others[0], tokens[10:47], []), *entries, StepEntry(others[1], tokens[3:8], []), StepEntry(others[2], [tokens[7]], [])]
            got.append(ex.step(entries).cpu().numpy())
        runs[name] = np.concatenate(got)
        assert runs[name].shape == held.shape and rel_error(runs[name], held) <= allowed
        ex.release(request)
    for name in ("beside decoding", "beside prompts"):
        assert rel_error(runs[name], runs["alone"]) <= allowed
    ex.cache.check_invariants()
