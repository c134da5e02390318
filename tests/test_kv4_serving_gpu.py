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


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_the_cache_holds_the_codes_of_the_rows_that_the_engine_appended(tmp_path, monkeypatch, dtype):
    """Bit by bit, every layer, portions and tokens: what `kv4_append` was given, in the slots that it was given."""
    import plain_kv4
    from tiny_inference_engine_b200 import StepEntry, StepRunner, load_model, make_cache, ops
    cfg = {**plain.TINY_D, "num_hidden_layers": 3}          # (fewer layers than are issued by one call)
    plain.write_model_dir(tmp_path, cfg, plain.random_weights(cfg, 6))
    model = load_model(tmp_path, dtype)
    cache, states = make_cache(model, page_size=8, num_pages=30, max_requests=4, kv_bits=4)
    runner = StepRunner(model, cache, 64, 4, 64, states=states, use_graphs=False)
    heads, dim = 2, 64
    want = [[np.full(tuple(t.shape), 0x3a, np.uint8 if t.dtype == torch.uint8 else np.uint16) for t in cache.layer_cache(e, True).kv4[:4]] for e in range(3)]
    for e in range(3):
        for t, fill in zip(cache.layer_cache(e, True).kv4[:4], want[e]):
            t.fill_(0x3a)
    where = {cache.layer_cache(e, True).kv4.k_codes.data_ptr(): e for e in range(3)}
    append = ops.kv4_append

    def recorded(k, v, slots, four):
        planes = want[where[four.k_codes.data_ptr()]]
        new = [part for pair in plain_kv4.quantise(*(x.float().cpu().numpy().reshape(-1, heads, dim) for x in (k, v))) for part in pair]
        for i, s in enumerate(slots.tolist()):
            if s >= 0:
                for plane, rows in zip(planes, new):
                    plane[s // 8, :, s % 8] = rows[i]
        append(k, v, slots, four)
    monkeypatch.setattr(ops, "kv4_append", recorded)
    rng = np.random.default_rng(2)
    a, b = (rng.integers(0, cfg["vocab_size"], n).tolist() for n in (60, 20))
    ra, rb = cache.new_request(), cache.new_request()
    assert cache.reserve(ra, 60) and cache.reserve(rb, 20)
    runner.run([StepEntry(ra, a[:50], 0, [49])])
    runner.run([StepEntry(ra, a[50:57], 50, [6]), StepEntry(rb, b[:17], 0, [16])])
    for i in range(3):
        runner.run([StepEntry(ra, [a[57 + i]], 57 + i, [0]), StepEntry(rb, [b[17 + i]], 17 + i, [0])])
    torch.cuda.synchronize()
    runner.check()
    for e in range(3):
        for t, w in zip(cache.layer_cache(e, True).kv4[:4], want[e]):
            assert np.array_equal(t.cpu().numpy().view(w.dtype), w), e
        assert (want[e][0] != 0x3a).any()


@pytest.mark.parametrize("ahead", [False, True])
def test_requests_that_are_preempted_are_computed_again(tmp_path, ahead):
    from tiny_inference_engine_b200 import SamplingParams, ServingConfig, load_engine
    cfg = {**plain.TINY_B, "num_hidden_layers": 4}
    plain.write_model_dir(tmp_path, cfg, plain.random_weights(cfg, 2))
    rng = np.random.default_rng(14)
    prompts = [rng.integers(0, cfg["vocab_size"], n).tolist() for n in (3, 17, 8, 25, 1, 11)]
    params = [SamplingParams(max_tokens=5 + 4 * i) for i in range(6)]
    eng = load_engine(tmp_path, dtype="float32", num_pages=9, page_size=8, policy="fcfs", kv_bits=4, serving=ServingConfig(16, 8, run_ahead=ahead))
    got = eng.generate_batch(prompts, params)
    while eng.has_work():
        eng.step()
    assert eng.stats().preemptions > 0 and eng.cache.num_free() == 9 and [len(t) for t in got] == [p.max_tokens for p in params]
    wide = load_engine(tmp_path, dtype="float32", num_pages=64, page_size=8, policy="fcfs", kv_bits=4, serving=ServingConfig(16, 8, run_ahead=ahead))
    # (a number on the border of two codes may fall otherwise when its product runs beside other rows: of six requests one at most)
    assert sum(x != y for x, y in zip(got, wide.generate_batch(prompts, params))) <= 1


def test_the_command_line_generates_what_the_engine_does(tmp_path, capsys):
    from tiny_inference_engine_b200 import SamplingParams, load_engine
    from tiny_inference_engine_b200.cli.main import main
    cfg = plain.TINY_D
    plain.write_model_dir(tmp_path, cfg, plain.random_weights(cfg, 9))
    want = load_engine(tmp_path, dtype="float32", kv_mem=4 << 20, kv_bits=4).generate([5, 6, 7], SamplingParams(max_tokens=12))
    assert main(["generate", "-m", str(tmp_path), "-p", "5 6 7", "--temp", "0", "--max-tokens", "12", "--dtype", "float32", "--kv-mem", "4M", "--kv-bits", "4"]) == 0
    out = capsys.readouterr()
    assert [int(t) for t in out.out.split()] == want
    cfg_bytes = 2 * 2 * 2 * 36 * 16                     # layers, keys and values, heads, bytes of a row of 64, tokens of a page
    assert f"pool {(4 << 20) // cfg_bytes} blocks" in out.err
