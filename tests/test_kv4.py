"""The operators of a cache in 4 bits, what runs without a GPU: the format's own properties, and every refusal."""
import numpy as np
import pytest
import torch

import plain_kv4 as plain
from tiny_inference_engine_b200 import ops
from tiny_inference_engine_b200.errors import InvalidArgument


def test_every_value_is_a_bfloat16_number_within_a_step():
    rng = np.random.default_rng(0)
    x = (rng.standard_normal((500, 96)) * np.exp(4 * rng.standard_normal((500, 1))) + rng.standard_normal((500, 1))).astype(np.float32)
    (c, w), _ = plain.quantise(x, x)
    v = plain.values(c, w, 96)
    assert np.array_equal(torch.tensor(v).to(torch.bfloat16).double().numpy(), v)
    s = ((w.astype(np.uint32) & 0xffe0) << 16).view(np.float32)
    assert (np.abs(v - x) <= np.repeat(s, 32, -1)[:, :96] * 1.0000001).all()
    # the step is less than 5/4 of what the range needs
    g = np.concatenate([x, np.zeros((500, 32), np.float32)], 1).reshape(500, 4, 32)
    assert (s <= 1.25 * (np.maximum(g.max(-1), 0) - np.minimum(g.min(-1), 0)) / 15 + 2.0 ** -100).all()


def test_quotients_by_a_step_tie_only_where_they_tie_exactly():
    """rint of the 32-bit quotient is rint of the exact one, for divisors of three significant bits."""
    rng = np.random.default_rng(1)
    s = (rng.integers(4, 8, 200000) * 2.0 ** rng.integers(-8, 8, 200000)).astype(np.float32)
    near = ((rng.integers(-15, 15, 200000) + 0.5) * s).astype(np.float32)
    for x in (near, np.nextafter(near, np.float32(np.inf)), np.nextafter(near, np.float32(-np.inf)), (s * rng.uniform(-15, 15, 200000)).astype(np.float32)):
        assert np.array_equal(np.rint(x / s).astype(np.float64), np.rint(x.astype(np.float64) / s.astype(np.float64)))


def cache(pages=3, kv_heads=2, page=4, head_dim=64):
    return ops.kv4_cache(pages, kv_heads, page, head_dim, device="cpu")


def i32(*x):
    return torch.tensor(x, dtype=torch.int32)


def refused(fn, *args, match=None, **kw):
    with pytest.raises(InvalidArgument, match=match):
        fn(*args, **kw)


def test_cache_sizes():
    c = cache(head_dim=96)
    assert c.k_codes.shape == (3, 2, 4, 64) and c.v_words.shape == (3, 2, 4, 4) and c.k_words.dtype == torch.int16
    for bad in ((0, 1, 1, 64), (1, 0, 1, 64), (1, 1, 0, 64), (1, 1, 1, 0), (1, 1, 1, 257), (2 ** 28, 1, 16, 64)):
        refused(ops.kv4_cache, *bad, device="cpu")


@pytest.mark.parametrize("fn", ["append", "read"])
def test_append_and_read_refuse(fn):
    def go(k, v, slots, c):
        return ops.kv4_append(k, v, slots, c) if fn == "append" else ops.kv4_read(c, slots, k, v)
    x, s = torch.zeros(3, 128), i32(0, 1, 2)
    refused(go, x, x, s, cache(), match="CUDA")                       # all right but for the device
    refused(go, x.half(), x.half(), s, cache(), match="float32 or bfloat16")
    refused(go, x, x.bfloat16(), s, cache(), match="alike")
    refused(go, x[:, :64], x[:, :64], s, cache())
    refused(go, x, x[:2], s, cache())
    refused(go, x[:1].expand(3, -1), x, s, cache(), match="overlap" if fn == "read" else "CUDA")      # (append only reads them)
    refused(go, torch.zeros(3, 256)[:, ::2], x, s, cache())
    refused(go, x, x, s[:2], cache(), match="slots")
    refused(go, x, x, s.long(), cache(), match="slots")
    c = cache()
    refused(go, x, x, s, c._replace(head_dim=300))
    refused(go, x, x, s, c._replace(head_dim=65))
    refused(go, x, x, s, c._replace(v_words=c.v_words[:2]))
    refused(go, x, x, s, c._replace(k_codes=c.k_codes.transpose(0, 1)))
    refused(go, x, x, s, c._replace(k_words=c.k_words.int()))


def test_attention_refuses():
    q, out, c = torch.zeros(2, 256), torch.zeros(2, 256), cache()
    start, lens, tables, work = i32(0, 1, 2), i32(3, 4), torch.zeros(2, 1, dtype=torch.int32), ops.kv4_workspace(4, 2, 64, device="cpu")
    good = dict(q=q, cache=c, out=out, query_start=start, context_lens=lens, block_tables=tables, q_heads=4, scale=0.1, max_context=4, workspace=work)
    for fn, extra in ((ops.attention_kv4_decode, dict(seq_list=i32(0, 1), n_list=2)), (ops.attention_kv4_prompt, dict(n_seqs=2, max_queries=1))):
        refused(fn, **good, **extra, match="CUDA")
        for bad in (dict(q=q.half(), out=out.half()), dict(out=out.bfloat16()), dict(q_heads=3), dict(q_heads=0), dict(q=q[:, :128]), dict(out=out[:1]),
                    dict(out=torch.zeros(2, 512)[:, ::2]), dict(query_start=start[:2]), dict(query_start=start.long()), dict(context_lens=lens.long()),
                    dict(block_tables=tables[:1]), dict(block_tables=tables[0]), dict(block_tables=torch.zeros(2, 2, dtype=torch.int32)[:, ::2]), dict(scale=0.0),
                    dict(scale=float("nan")), dict(max_context=-1), dict(window=-1), dict(workspace=ops.Kv4Workspace(work.scratch[:9], work.counters)),
                    dict(workspace=ops.Kv4Workspace(work.scratch, work.counters[:9])), dict(cache=c._replace(head_dim=0))):
            refused(fn, **{**good, **extra, **bad})
    refused(ops.attention_kv4_decode, **good, seq_list=i32(0), n_list=2, match="seq_list")
    refused(ops.attention_kv4_decode, **good, seq_list=torch.tensor([0, 1]), n_list=2, match="seq_list")
    refused(ops.attention_kv4_decode, **good, seq_list=i32(0, 1), n_list=-1)
    refused(ops.attention_kv4_prompt, **good, n_seqs=3, max_queries=1)
    refused(ops.attention_kv4_prompt, **good, n_seqs=2, max_queries=-1)
    refused(ops.kv4_workspace, 3, 2, 64, device="cpu")
    refused(ops.Kv4Workspace, work.scratch.double(), work.counters)
    refused(ops.Kv4Workspace, work.scratch[::2], work.counters)
    refused(ops.Kv4Workspace, work.scratch[1:], work.counters)
    refused(ops.Kv4Workspace, work.scratch, work.counters.long())


def test_step_tables_refuse():
    good = dict(requests=i32(0, 2), counts=i32(1, 1), lens=i32(0, 0, 0), tables=torch.zeros(3, 5, dtype=torch.int32), free_pages=i32(0, 1, 2), free_count=i32(3),
                page_size=4, arrays=ops.step_arrays(2, 2, 5, device="cpu"))
    refused(ops.step_tables, **good, match="CUDA")
    for bad in (dict(requests=i32(0)), dict(requests=torch.tensor([0, 2])), dict(counts=i32(1)), dict(lens=i32(0, 0)), dict(free_count=i32(3, 3)),
                dict(tables=torch.zeros(5, 3, dtype=torch.int32).T), dict(page_size=0), dict(arrays=ops.step_arrays(3, 2, 5, device="cpu")),
                dict(arrays=ops.step_arrays(2, 2, 6, device="cpu")), dict(arrays=good["arrays"]._replace(slots=torch.zeros(2))),
                dict(arrays=good["arrays"]._replace(positions=i32(0)))):
        refused(ops.step_tables, **{**good, **bad})
    good.pop("arrays"), good.pop("counts")
    refused(ops.release_tables, **good, status=i32(0), match="CUDA")
    refused(ops.release_tables, **good, status=i32(0, 0))
    for bad in ((-1, 1, 1), (1, -1, 1), (1, 1, 0)):
        refused(ops.step_arrays, *bad, device="cpu")


def test_cache_manager_counts_the_bytes_of_4_bits():
    from tiny_inference_engine_b200.cache import CacheManager
    from tiny_inference_engine_b200.errors import UnsupportedError
    from tiny_inference_engine_b200.parts.base import CacheNeed
    needs = [CacheNeed("full", 8, 128)] * 3 + [CacheNeed("window", 2, 96, 64)]
    wide = CacheManager(needs, 16, num_pages=5, dtype=torch.bfloat16)
    four = CacheManager(needs, 16, num_pages=5, dtype=torch.bfloat16, kv_bits=4)
    assert wide.bytes_per_page == 16 * 2 * 2 * (3 * 8 * 128 + 2 * 96)
    assert four.bytes_per_page == 16 * 2 * (3 * 8 * 72 + 2 * 72)              # 64 bytes of codes and 8 of words; 96 is padded to 128
    made = CacheManager(needs, 16, num_pages=5, dtype=torch.bfloat16, device="cpu", kv_bits=4)
    assert sum(t.numel() * t.element_size() for pair in made.storage for t in pair) == 5 * four.bytes_per_page
    view = made.layer_cache(2, True)
    assert view.k is None and view.kv4.head_dim == 128 and tuple(view.kv4.k_codes.shape) == (5, 8, 16, 64) and tuple(view.kv4.v_words.shape) == (5, 8, 16, 4)
    view.kv4.v_codes.fill_(7)                          # the planes are apart
    assert int((made.storage[0][0] == 7).sum()) == view.kv4.v_codes.numel() and int(made.layer_cache(2, True).kv4.k_codes.sum()) == 0
    for need in (CacheNeed("full", 1, 64, value_dim=-1), CacheNeed("full", 1, 64, value_dim=32), CacheNeed("full", 1, 512), CacheNeed("window", 1, 64, 8, keep_first=4)):
        with pytest.raises(UnsupportedError):
            CacheManager([need], 16, num_pages=5, kv_bits=4)
    refused(CacheManager, needs, 16, num_pages=5, kv_bits=8, match="kv_bits")


def test_designs_whose_mixers_know_no_4_bits_are_refused():
    import plain_misudra
    from tiny_inference_engine_b200 import make_cache
    from tiny_inference_engine_b200.config import misudra_spec, parse_misudra_config
    from tiny_inference_engine_b200.errors import UnsupportedError
    from tiny_inference_engine_b200.parts.model import Model
    cfg = plain_misudra.make_config([plain_misudra.latent_layer(mlp=plain_misudra.dense())])
    with pytest.raises(UnsupportedError, match="4 bits"):
        make_cache(Model(misudra_spec(parse_misudra_config(cfg)), torch.float32), num_pages=4, device="cpu", kv_bits=4)


def test_queries_and_keys_in_place_refuse():
    x, w, pos = torch.zeros(3, 256), torch.ones(64), torch.zeros(3, dtype=torch.int32)
    for bad, why in (((x[:, :100], w, w, pos), "narrow"), ((x, w[:32], w, pos), "weights"), ((x, w, w.double(), pos), "weights"), ((x, w, w, pos[:2]), "positions"),
                     ((x, w, w, pos.long()), "positions"), ((x, w, w, pos), "CUDA")):
        refused(ops.qk_norm_rope, *bad[:3], 1e-6, 1e-6, None, bad[3], 2, 1, 64, match=why)
    refused(ops.qk_norm_rope, x, w, w, 1e-6, 1e-6, w.double(), pos, 2, 1, 64, match="inv_freq")
