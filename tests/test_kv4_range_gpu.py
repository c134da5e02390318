"""Attention over a cache in 4 bits sees what `kv4_read` gives over the whole range of steps that the format has, 2^-100 to about 2^117, side by side in
a tile, a row of a tile and a token. The batches of test_kv4_gpu.py, whose words get other exponents: a step times a power of two is what the
same numbers times that power would have got. Keys' powers are taken back in the queries, so that scores stay what they were; tolerances are that file's with M,
the largest value that a row's output could be made of, taken for each dimension on its own: dimensions are summed apart."""
import numpy as np
import pytest
import torch

import plain_kv4 as plain
from test_kv4_gpu import DT, Batch, cuda, planes, rounded
from tiny_inference_engine_b200 import ops
from tiny_inference_engine_b200.ops import kv4

pytestmark = pytest.mark.gpu
LEAST = (127 - 100) << 7           # the word of a step of 2^-100: of groups of zeros, which have no larger one


def rescaled(b, page, key_powers, value_powers):
    """b with key head h times 2^key_powers[h] (its queries divided by that) and a value group's step times 2^ one of value_powers, at random."""
    rng = np.random.default_rng(len(value_powers))
    _, kw, _, vw = planes(b.cache)
    group = b.heads // b.kv_heads
    kp = np.array(key_powers)[np.arange(b.kv_heads) % len(key_powers)]
    vp = rng.choice(value_powers, vw.shape)
    for words, power, fill in ((kw, kp[None, :, None, None], 0x7f81), (vw, vp, 0x4000)):
        moved = np.where((words != fill) & ((words & 0xffe0) != LEAST) & (words != 0), words.astype(np.int64) + (power << 7), words)
        assert moved.min() >= 0 and moved.max() <= 0x7fff
        words[...] = moved.astype(np.uint16)
    b.cache.k_words.copy_(cuda(kw.view(np.int16), torch.int16))
    b.cache.v_words.copy_(cuda(vw.view(np.int16), torch.int16))
    q = rounded(b.q * (2.0 ** -kp.astype(np.float64))[np.arange(b.heads) // group][None, :, None], b.dtype)
    b.qt[:, :b.heads * b.head_dim] = cuda(q.reshape(len(q), -1), DT[b.dtype])
    kc, kw, vc, vw = planes(b.cache)
    tables = b.args[2].cpu().numpy()
    b.most = np.zeros(b.want.shape)
    for i, c in enumerate(b.contexts):
        if not c:
            continue
        at = tables[i, np.arange(c) // page], slice(None), np.arange(c) % page
        kx, vx = (plain.values(codes[at], words[at], b.head_dim) for codes, words in ((kc, kw), (vc, vw)))
        first, last = b.start[i], b.start[i + 1]
        pos = np.arange(c - (last - first), c)
        for h in range(b.heads):
            b.want[first:last, h] = plain.attention(q[first:last, h].astype(np.float64), kx[:, h // group], vx[:, h // group], pos, b.scale, b.window)
            b.most[first:last, h] = np.abs(vx[:, h // group]).max(0)
    return b


POWERS = [([-97], [-97]), ([100], [115]), ([0], [15, 25, 26, 27]), ([-60, 0, 70], [-60, 0]), ([30, -97, 100], [-97, -40, 0, 58, 115])]


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("keys,values", POWERS)
@pytest.mark.parametrize("contexts,heads,kv_heads,head_dim,page", [([33, 1, 257], 8, 2, 128, 16), ([700, 45], 6, 3, 64, 8), ([130], 7, 1, 80, 12), ([190, 9], 5, 5, 192, 3),
                                                                  ([2500], 40, 4, 256, 16)])
def test_tokens(dtype, keys, values, contexts, heads, kv_heads, head_dim, page):
    b = rescaled(Batch(head_dim, contexts, [1] * len(contexts), heads, kv_heads, head_dim, page, dtype), page, keys, values)
    b.check(b.decode())


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("keys,values", POWERS)
@pytest.mark.parametrize("head_dim,long", [(64, False), (128, False), (256, False), (64, True), (96, True), (128, True), (192, True), (256, True)])
def test_portions(monkeypatch, dtype, keys, values, head_dim, long):
    if long:
        monkeypatch.setattr(kv4, "UMMA_GROUPS", 0)
    queries = [130, 40] if long else [9, 33]
    b = rescaled(Batch(head_dim + 1, [300, 70], queries, 8, 2, head_dim, 16, dtype, window=90, pad=8 if long else 5), 16, keys, values)
    b.check(b.prompt(), one_term=True, truncated=long)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_what_is_appended_is_what_attention_sees(dtype):
    """One key a sequence: its value comes out as `kv4_read` gives it, from the least to the largest numbers that a cache holds."""
    powers = np.arange(-104, 120)
    n, dim = len(powers), 64
    rng = np.random.default_rng(2)
    x = (1.0 + rng.random((n, dim))) * np.sign(rng.standard_normal((n, dim))) * 2.0 ** (powers[:, None] - 1.0)
    x = rounded(x, dtype)
    cache = ops.kv4_cache(n, 1, 1, dim)
    slots = cuda(np.arange(n))
    keys = torch.zeros(n, dim, dtype=DT[dtype], device="cuda")
    ops.kv4_append(keys, cuda(x, DT[dtype]), slots, cache)
    k, v, out = (torch.empty_like(keys) for _ in range(3))
    ops.kv4_read(cache, slots, k, v)
    q = torch.ones_like(keys)
    args = q, cache, out, cuda(np.arange(n + 1)), cuda(np.ones(n)), slots.view(n, 1)
    ops.attention_kv4_decode(*args, 1, 1.0, slots, n, 1, ops.kv4_workspace(1, 1, dim))
    torch.cuda.synchronize()
    # a weight that is 1 but for the row sum's quotient: a rounding of the quotient and one of the product, 2^-24 each
    limit = v.double().abs() * (2.0 ** -23 if dtype == "float32" else 2.0 ** -8)
    assert bool(((out.double() - v.double()).abs() <= limit).all()) and bool((v[-1] != 0).all())
