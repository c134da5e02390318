"""The engine over a cache in 4 bits (`kv_bits=4`), against the plain implementation over the values that the engine's cache holds.

The engine's keys and values reach the codes with other rounding errors than plain ones (order of sums, bfloat16 activations), so a number
near the border of two codes may fall to the other side and move by a step, and with it every later row of every later layer. So two things are
held: the cached values are the plain codes of the plain keys and values, but for few numbers that are a step or so off; and logits are, within
conftest.TOL, those of the plain model whose attention reads the very values that are in the cache."""
import numpy as np
import pytest
import torch

import plain_kv4
import plain_qwen3 as plain
from conftest import assert_logits_close

pytestmark = pytest.mark.gpu


def cached_values(cache, req, n):
    """Per layer what the cache holds for the request's first n tokens: (keys, values), float32 [n, kv heads * head size]."""
    from tiny_inference_engine_b200 import ops
    slots = torch.as_tensor(cache.slots(req, 0, 0, n)).cuda()
    out = []
    for entry in range(len(cache.groups[0].entries)):
        four = cache.layer_cache(entry, False).kv4
        k, v = (torch.empty(n, four.kv_heads * four.head_dim, device="cuda") for _ in range(2))
        ops.kv4_read(four, slots, k, v)
        out.append((k.cpu().numpy(), v.cpu().numpy()))
    return out


def forward_over(monkeypatch, w, cfg, tokens, values):
    """The plain model's logits with each layer's attention over the given keys and values; and the plain keys and values of every layer."""
    attention, own, at = plain.causal_attention, [], iter(values)

    def over(q, k, v, heads, kv_heads, dim, window=0):
        own.append((k, v))
        return attention(q, *next(at), heads, kv_heads, dim, window)
    with monkeypatch.context() as m:
        m.setattr(plain, "causal_attention", over)
        return plain.forward(w, cfg, tokens), own


def check(monkeypatch, w, cfg, cache, req, tokens, got, rows, dtype, what):
    """got: the engine's logits of `rows` of the request's tokens, all of which are in the cache."""
    values = cached_values(cache, req, len(tokens))
    want, own = forward_over(monkeypatch, w, cfg, tokens, values)
    assert_logits_close(got, want[rows], dtype, what)
    kv_heads, dim = cfg["num_key_value_heads"], cfg["head_dim"]
    for (k, v), held in zip(own, values):
        for (codes, words), have in zip(plain_kv4.quantise(*(x.astype(np.float32).reshape(len(tokens), kv_heads, dim) for x in (k, v))), held):
            have = have.reshape(len(tokens), kv_heads, dim)
            off = np.abs(plain_kv4.values(codes, words, dim) - have)
            # float32 moves numbers within about 1e-5 steps of a border; bfloat16 activations, off by a percent of numbers that are up to 8 steps
            # from zero, about one in ten, and where a scale itself falls otherwise (by a quarter at most) all of its group
            assert (off > 0).mean() <= (0.01 if dtype == "float32" else 0.4), what
            assert (off <= 0.5 * np.abs(have).max(-1, keepdims=True) + 1e-6).all(), what


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("cfg,page", [(plain.TINY_A, 16), (plain.TINY_B, 8), (plain.TINY_C, 12), (plain.TINY_D, 16), (plain.TINY_E, 64)])
def test_logits_however_the_work_is_cut(tmp_path, monkeypatch, cfg, page, dtype):
    from tiny_inference_engine_b200 import StepEntry, StepRunner, load_model, make_cache
    cfg = {**cfg, "num_hidden_layers": 5}           # (alike layers: those from the third on are issued by one call)
    w = plain.random_weights(cfg, 3)
    plain.write_model_dir(tmp_path, cfg, w)
    norm = plain.normalise_config(cfg)
    rng = np.random.default_rng(5)
    a, b = (rng.integers(0, cfg["vocab_size"], n).tolist() for n in (150, 41))
    model = load_model(tmp_path, dtype)
    cache, states = make_cache(model, page_size=page, num_pages=-(-150 // page) + -(-41 // page) + 2, max_requests=4, kv_bits=4)
    for part in cache.storage[0]:
        part.fill_(0x53)                            # pages hold whatever was there
    runner = StepRunner(model, cache, 160, 4, 200, states=states)
    wq = {k: (plain.round_bf16(v) if dtype == "bfloat16" and v.ndim == 2 else v) for k, v in w.items()}

    def logits(entries):
        return runner.run(entries).float().cpu().numpy().copy()

    def same(req, tokens, got, first, what):
        check(monkeypatch, wq, norm, cache, req, tokens, got, slice(first, None), dtype, what)

    ra = cache.new_request()
    assert cache.reserve(ra, 150)
    same(ra, a, logits([StepEntry(ra, a, 0, list(range(150)))]), 0, "whole")
    cache.release(ra)
    ra, rb = cache.new_request(), cache.new_request()
    assert cache.reserve(ra, 150) and cache.reserve(rb, 41)
    same(ra, a[:67], logits([StepEntry(ra, a[:67], 0, list(range(67)))]), 0, "a portion")
    got = logits([StepEntry(ra, a[67:130], 67, list(range(63))), StepEntry(rb, b[:30], 0, list(range(30)))])
    same(ra, a[:130], got[:63], 67, "the next portion")
    same(rb, b[:30], got[63:], 0, "a portion of another")
    for i in range(11):                             # tokens one by one, of both
        got = logits([StepEntry(ra, [a[130 + i]], 130 + i, [0]), StepEntry(rb, [b[30 + i]], 30 + i, [0])])
        same(ra, a[:131 + i], got[:1], 130 + i, f"token {i}")
        same(rb, b[:31 + i], got[1:], 30 + i, f"token {i} of another")
    assert runner.graph_replays > 5
    same(ra, a, logits([StepEntry(ra, a[141:], 141, list(range(9)))]), 141, "a short portion")
    torch.cuda.synchronize()
    runner.check()


def test_generation_batched_and_alone_and_the_bytes_of_the_cache(tmp_path):
    from tiny_inference_engine_b200 import SamplingParams, ServingConfig, load_engine
    cfg = {**plain.TINY_D, "num_hidden_layers": 4}
    plain.write_model_dir(tmp_path, cfg, plain.random_weights(cfg, 0))
    wide = load_engine(tmp_path, kv_mem=4 << 20)
    eng = load_engine(tmp_path, kv_mem=4 << 20, kv_bits=4, serving=ServingConfig(64, 8))
    assert eng.cache.bytes_per_page * 128 == wide.cache.bytes_per_page * 36       # 4.5 bits a value for 16
    assert eng.cache.num_pages > 3.5 * wide.cache.num_pages
    rng = np.random.default_rng(1)
    prompts = [rng.integers(0, cfg["vocab_size"], n).tolist() for n in (5, 40, 70, 1, 130, 17)]
    params = [SamplingParams(max_tokens=12, temperature=0.7, seed=i) for i in range(len(prompts))]
    alone = [eng.generate(p, q) for p, q in zip(prompts, params)]
    together = eng.generate_batch(prompts, params)
    # a number on the border of two codes may fall otherwise when its product runs beside other rows: of six requests one at most
    assert sum(x != y for x, y in zip(alone, together)) <= 1 and all(len(t) == 12 for t in together)
    assert eng.cache.num_free() == eng.cache.num_pages
