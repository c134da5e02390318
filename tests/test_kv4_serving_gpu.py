"""The engine over a cache in 4 bits where its steps are filled up, cut short or planned again."""
import numpy as np
import pytest
import torch

import plain_qwen3 as plain
from test_kv4_engine_gpu import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_padded_decode_steps_with_small_pages(tmp_path, monkeypatch, dtype):
    """Three requests in a captured step of four: the fourth sequence has no keys, and its table row is the last of the index buffer, in which
    whatever else it held stands behind."""
    from tiny_inference_engine_b200 import StepEntry, StepRunner, load_model, make_cache
    cfg = {**plain.TINY_A, "num_hidden_layers": 4}
    w = plain.random_weights(cfg, 3)
    plain.write_model_dir(tmp_path, cfg, w)
    norm = plain.normalise_config(cfg)
    model = load_model(tmp_path, dtype)
    cache, states = make_cache(model, page_size=8, num_pages=24, max_requests=4, kv_bits=4)
    runner = StepRunner(model, cache, 64, 4, 64, states=states)
    runner._dev.fill_(-1)
    wq = {k: (plain.round_bf16(v) if dtype == "bfloat16" and v.ndim == 2 else v) for k, v in w.items()}
    rng = np.random.default_rng(6)
    said = [rng.integers(0, cfg["vocab_size"], 30).tolist() for _ in range(3)]
    held = [13, 1, 20]
    reqs = [cache.new_request() for _ in range(3)]
    for req, tokens, n in zip(reqs, said, held):
        assert cache.reserve(req, 30)
        runner.run([StepEntry(req, tokens[:n], 0, [n - 1])])
    for step in range(9):
        got = runner.run([StepEntry(req, [tokens[n + step]], n + step, [0]) for req, tokens, n in zip(reqs, said, held)]).float().cpu().numpy().copy()
        torch.cuda.synchronize()
        runner.check()
        for i, (req, tokens, n) in enumerate(zip(reqs, said, held)):
            check(monkeypatch, wq, norm, cache, req, tokens[:n + step + 1], got[i:i + 1], slice(n + step, None), dtype, f"request {i}, step {step}")
    assert runner.graph_replays >= 8


@pytest.mark.parametrize("page,pages", [(5, 7), (2, 15), (3, 11)])
def test_pages_whose_planes_of_words_are_no_whole_16_bytes(tmp_path, monkeypatch, page, pages):
    from tiny_inference_engine_b200 import StepEntry, StepRunner, load_model, make_cache
    cfg = {**plain.TINY_B, "num_hidden_layers": 3}
    w = plain.random_weights(cfg, 4)
    plain.write_model_dir(tmp_path, cfg, w)
    model = load_model(tmp_path, "float32")
    cache, states = make_cache(model, page_size=page, num_pages=pages, max_requests=2, kv_bits=4)
    runner = StepRunner(model, cache, 64, 2, 64, states=states)
    tokens = np.random.default_rng(8).integers(0, cfg["vocab_size"], 29).tolist()
    req = cache.new_request()
    assert cache.reserve(req, 29)
    runner.run([StepEntry(req, tokens[:25], 0, [24])])
    for i in range(25, 29):
        got = runner.run([StepEntry(req, [tokens[i]], i, [0])]).float().cpu().numpy().copy()
        torch.cuda.synchronize()
        runner.check()
        check(monkeypatch, w, plain.normalise_config(cfg), cache, req, tokens[:i + 1], got, slice(i, None), "float32", f"token {i}")
