"""The operators of a cache in 4 bits on the GPU, against numpy in 64 bits (plain_kv4.py).

Tolerances, derived. What the cache holds is defined exactly, so codes, words and tables are compared bit by bit. Attention: the products'
operands are exact (values of the cache are bfloat16 numbers, queries enter with all their bits), so what is off is, for a row whose values
are at most M in magnitude (the output is a convex sum of them):
  bfloat16 rows   the output's rounding, half a step: eps / 2 = 2^-8 of |o| at most, the weights as two bfloat16 terms (2^-16 relative, times M), and the sums of
                  the float products: a score of terms whose magnitudes add up to A is off by about 2^-22 A (the tensor cores add with
                  a few bits more than a float of the largest term), and exp turns that into as much of a weight. Below, A <= 64 in the
                  exponent's units, so 64 * 2^-22 = 2^-16, times M again for weights and row sum each: |o| 2^-8 + M 2^-14.
  float rows      three terms (2^-24), the sums as above: A <= 64: M (2 * 2^-16 + 2^-20), held to M 2^-15 + |o| 2^-23.
The portions' tcgen05 kernel rounds weights to one bfloat16 term: a weight is off by eps / 2 = 2^-8 of itself,
the output by 2^-8 M more."""
import numpy as np
import pytest
import torch

import plain_kv4 as plain
from tiny_inference_engine_b200 import ops
from tiny_inference_engine_b200.errors import TieError
from tiny_inference_engine_b200.ops import gemm_select, kv4

pytestmark = pytest.mark.gpu
NP = {"float32": np.float32, "bfloat16": np.float32}
DT = {"float32": torch.float32, "bfloat16": torch.bfloat16}


def cuda(x, dtype=torch.int32):
    return torch.as_tensor(np.ascontiguousarray(x)).to(dtype).cuda()


def rounded(x, dtype):
    """float32 numpy values that the type can hold."""
    return torch.tensor(x, dtype=torch.float32).to(DT[dtype]).float().numpy()


def planes(cache):
    torch.cuda.synchronize()
    return [t.cpu().numpy() if t.dtype == torch.uint8 else t.cpu().numpy().view(np.uint16) for t in cache[:4]]


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("T,kv_heads,head_dim,page,strided", [(1, 1, 64, 16, False), (7, 8, 128, 16, True), (33, 3, 96, 12, True), (5, 2, 80, 8, False),
                                                              (130, 1, 256, 1, True), (9, 5, 192, 5, False), (6, 2, 7, 4, True), (3, 3, 33, 16, False),
                                                              (700, 4, 128, 64, True)])
def test_append_and_read(dtype, T, kv_heads, head_dim, page, strided):
    rng = np.random.default_rng(T * 31 + head_dim)
    width = kv_heads * head_dim
    k, v = (rounded(rng.standard_normal((T, width)) * np.exp(rng.standard_normal(width)), dtype) for _ in range(2))
    k[0, :] = 0.0                                    # a group of zeros
    if T > 2:
        k[1] = np.abs(k[1])                          # one-sided groups
        v[1] = -np.abs(v[1])
        v[2] *= np.float32(1e-30)                    # small ones, below the least step
        k[2] *= np.float32(1e-36)
        k, v = rounded(k, dtype), rounded(v, dtype)
    pages = -(-T // page) + 2
    slots = rng.permutation(pages * page)[:T].astype(np.int32)
    slots[T // 2] = -1 if T > 1 else slots[0]
    cache = ops.kv4_cache(pages, kv_heads, page, head_dim)
    for t in cache[:4]:
        t.fill_(77)                                  # what is not written stays
    if strided:
        rows = torch.zeros(T, 2 * width + 3, dtype=DT[dtype], device="cuda")
        rows[:, 1:1 + width], rows[:, 2 + width:2 + 2 * width] = cuda(k, DT[dtype]), cuda(v, DT[dtype])
        kt, vt = rows[:, 1:1 + width], rows[:, 2 + width:2 + 2 * width]
    else:
        kt, vt = cuda(k, DT[dtype]), cuda(v, DT[dtype])
    ops.kv4_append(kt, vt, cuda(slots), cache)
    want = [np.full(t.shape, 77, np.uint8 if t.dtype == torch.uint8 else np.uint16) for t in cache[:4]]
    (kc, kw), (vc, vw) = plain.quantise(k.reshape(T, kv_heads, head_dim), v.reshape(T, kv_heads, head_dim))
    for i, s in enumerate(slots):
        if s >= 0:
            for plane, new in zip(want, (kc, kw, vc, vw)):
                plane[s // page, :, s % page] = new[i]
    for got, w in zip(planes(cache), want):
        assert np.array_equal(got, w)
    # and out again: exactly what the codes stand for; rows without a slot stay
    ko, vo = torch.full((T, width + 8), 5.0, dtype=DT[dtype], device="cuda"), torch.full((T, width), 5.0, dtype=DT[dtype], device="cuda")
    ops.kv4_read(cache, cuda(slots), ko[:, 8:], vo)
    for out, (c, w) in ((ko[:, 8:], (kc, kw)), (vo, (vc, vw))):
        expect = plain.values(c, w, head_dim).reshape(T, width)
        expect[slots < 0] = 5.0
        assert np.array_equal(out.float().cpu().numpy().astype(np.float64), expect)
    assert (ko[:, :8] == 5.0).all()
    # every value is within a step of what went in
    s = ((kw.astype(np.uint32) & 0xffe0) << 16).view(np.float32)
    err = np.abs(plain.values(kc, kw, head_dim) - k.reshape(T, kv_heads, head_dim))
    assert (err <= np.repeat(s, 32, -1)[..., :head_dim] * 1.0000001 + 2.0 ** -100).all()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("step", [1.0, 1.25, 1.75 * 2.0 ** 40, 2.0 ** -90])
def test_append_of_halves_that_round_up_at_both_ends(dtype, step):
    """The least -7.5 steps, the largest 7.5: z is 8 and the largest would be code 16. Halves and steps between them, in every place of a group."""
    rng = np.random.default_rng(3)
    x = (rng.integers(-15, 16, (64, 2, 80)) / 2 * step).astype(np.float32)
    for t in range(64):
        x[t, :, t % 32::32] = 7.5 * step
        x[t, :, (t + 1 + t // 32) % 32::32] = -7.5 * step
    cache = ops.kv4_cache(4, 2, 16, 80)
    ops.kv4_append(cuda(x.reshape(64, -1), DT[dtype]), cuda(-x.reshape(64, -1), DT[dtype]), cuda(np.arange(64)), cache)
    (kc, kw), (vc, vw) = plain.quantise(x, -x)
    order = lambda t: t.cpu().numpy().transpose(0, 2, 1, 3).reshape(64, 2, -1)
    assert np.array_equal(order(cache.k_codes), kc) and np.array_equal(order(cache.v_codes), vc)
    assert np.array_equal(order(cache.k_words), kw) and np.array_equal(order(cache.v_words), vw)
    top = np.stack([kc & 15, kc >> 4], -1).reshape(64, 2, -1)
    assert (top[np.arange(64), :, np.arange(64) % 32] == 15).all()


def test_append_marks_numbers_that_are_not_finite():
    T, heads, dim, page = 6, 2, 96, 4
    rng = np.random.default_rng(0)
    k, v = (rng.standard_normal((T, heads, dim)).astype(np.float32) for _ in range(2))
    k[0, 0, 5], k[1, 1, 95], v[2, 0, 0], v[3, 1, 50], k[4, 0, 3] = np.nan, np.inf, -np.inf, 2.0 ** 120, 1.3e36
    cache = ops.kv4_cache(2, heads, page, dim)
    slots = np.arange(T).astype(np.int32)
    ops.kv4_append(cuda(k.reshape(T, -1), torch.float32), cuda(v.reshape(T, -1), torch.float32), cuda(slots), cache)
    got = planes(cache)
    for plane, (c, w) in zip((got[:2], got[2:]), plain.quantise(k, v)):
        for x, y in zip(plane, (c, w)):
            assert np.array_equal(x[slots // page, :, slots % page], y)
    assert (got[1][0, 0, 0] == 0x7fc0).all() and (got[3][0, 0, 0] == 0).all()          # the head with a NaN
    assert (got[1][0, 1, 0] != 0x7fc0).all()                                           # its neighbour
    out = [torch.empty(T, heads * dim, device="cuda") for _ in range(2)]
    ops.kv4_read(cache, cuda(slots), *out)
    ko, vo = (o.cpu().numpy().reshape(T, heads, dim) for o in out)
    marked = np.zeros((T, heads), bool)
    marked[[0, 1, 2, 3], [0, 1, 0, 1]] = True
    assert np.isnan(ko[marked]).all() and (vo[marked] == 0).all() and np.isfinite(ko[~marked]).all() and np.isfinite(vo).all()


def test_slots_outside_of_the_cache_write_nothing():
    cache = ops.kv4_cache(2, 1, 4, 64)
    x = torch.ones(3, 64, device="cuda")
    ops.kv4_append(x, x, cuda([8, 2, 2 ** 31 - 1]), cache)
    torch.cuda.synchronize()
    with pytest.raises(TieError, match="slot"):
        gemm_select.check_status()
    assert int((cache.k_codes != 0).sum()) == 32 and bool((cache.k_codes[0, 0, 2] != 0).all())
    out = torch.full((1, 64), 3.0, device="cuda")
    ops.kv4_read(cache, cuda([9]), out, out.clone())
    torch.cuda.synchronize()
    with pytest.raises(TieError, match="slot"):
        gemm_select.check_status()
    assert bool((out == 3.0).all())


class Batch:
    """Sequences with random keys and values in a cache, their queries, and the answer in 64 bits."""

    def __init__(self, seed, contexts, queries, heads, kv_heads, head_dim, page, dtype, window=0, loud=1.0, nan_at=(), pad=5):
        rng = np.random.default_rng(seed)
        self.heads, self.kv_heads, self.head_dim, self.window, self.dtype = heads, kv_heads, head_dim, window, dtype
        n, T = len(contexts), sum(queries)
        pages = [-(-c // page) for c in contexts]
        ids = rng.permutation(sum(pages) + 2)
        columns = max(max(pages), 1) + 1
        tables = np.zeros((n, columns), np.int32)
        at = 0
        for i, p in enumerate(pages):
            tables[i, :p] = ids[at:at + p]
            at += p
        self.cache = ops.kv4_cache(sum(pages) + 2, kv_heads, page, head_dim)
        for words in (self.cache.k_words, self.cache.v_words):
            words.fill_(0x7f81 if words is self.cache.k_words else 0x4000)       # what no token of this batch wrote: keys of NaN, values of 2 (code - z)
        self.cache.k_codes.fill_(0x53)
        self.cache.v_codes.fill_(0xa7)
        self.q = rounded(rng.standard_normal((T, heads, head_dim)) * loud, dtype)
        self.scale = head_dim ** -0.5
        self.want = np.zeros((T, heads, head_dim))
        self.most = np.zeros((T, heads, 1))
        self.start = np.concatenate([[0], np.cumsum(queries)]).astype(np.int32)
        for i, c in enumerate(contexts):
            k, v = (rounded(rng.standard_normal((c, kv_heads, head_dim)), "bfloat16") for _ in range(2))
            for s, token in nan_at:
                if s == i:
                    v[token, 0, 0] = np.nan
            if c:
                slots = (tables[i, np.arange(c) // page] * page + np.arange(c) % page).astype(np.int32)
                ops.kv4_append(cuda(k.reshape(c, kv_heads * head_dim), torch.float32), cuda(v.reshape(c, kv_heads * head_dim), torch.float32), cuda(slots), self.cache)
            (kc, kw), (vc, vw) = plain.quantise(k, v)
            kx, vx = plain.values(kc, kw, head_dim), plain.values(vc, vw, head_dim)
            a, b = self.start[i], self.start[i + 1]
            pos = np.arange(c - queries[i], c)
            for h in range(heads):
                kv = h * kv_heads // heads
                self.want[a:b, h] = plain.attention(self.q[a:b, h].astype(np.float64), kx[:, kv], vx[:, kv], pos, self.scale, window)
                self.most[a:b, h] = np.abs(vx[:, kv]).max() if c else 0.0
        self.contexts, self.queries = contexts, queries
        self.args = (cuda(self.start), cuda(np.array(contexts, np.int32)), cuda(tables))
        self.work = ops.kv4_workspace(heads, kv_heads, head_dim)
        wide = torch.zeros(T, heads * head_dim + pad, dtype=DT[dtype], device="cuda")
        wide[:, :heads * head_dim] = cuda(self.q.reshape(T, -1), DT[dtype])
        self.qt = wide                                      # rows of a wider product's output
        self.out = torch.full((T, heads * head_dim), 9.0, dtype=DT[dtype], device="cuda")

    def decode(self, seqs=None, max_context=None):
        seqs = list(range(len(self.contexts))) if seqs is None else seqs
        ops.attention_kv4_decode(self.qt, self.cache, self.out, *self.args, self.heads, self.scale, cuda(seqs), len(seqs),
                                 max(self.contexts) if max_context is None else max_context, self.work, window=self.window)
        return self.answer()

    def prompt(self, n=None, max_queries=None):
        n = len(self.contexts) if n is None else n
        ops.attention_kv4_prompt(self.qt, self.cache, self.out, *self.args, n, max_queries or max(self.queries), self.heads, self.scale, max(self.contexts), self.work,
                                 window=self.window)
        return self.answer()

    def answer(self):
        torch.cuda.synchronize()
        gemm_select.check_status()
        assert int(self.work.counters.abs().sum()) == 0
        return self.out.float().cpu().numpy().astype(np.float64).reshape(self.want.shape)

    def check(self, got, rows=slice(None), one_term=False, truncated=False):
        """`truncated`: sums on tcgen05, whose every step may cut a unit of the running sum's last place instead of half a one. Of the scores (three
        terms, head_dim / 16 steps each, 24 for 128) by |q| |k| scale, here below 19, times 2^-23 each: the weights are off by 2^-13 with their sum.
        Of the values 3 keys / 16 steps, 206 for 1,100 keys: 2^-15. Together below M 2^-12."""
        want, most = self.want[rows], self.most[rows]
        if self.dtype == "float32":
            limit = most * 2.0 ** (-12 if truncated else -15) + np.abs(want) * 2.0 ** -23
        else:
            limit = np.abs(want) * 2.0 ** -8 + most * (2.0 ** -14 + (2.0 ** -8 if one_term else 0.0))
        assert np.array_equal(np.isnan(got[rows]), np.isnan(want))
        off = np.nan_to_num(np.abs(got[rows] - want) - limit * 1.001, nan=-1.0)
        assert off.max() <= 0, f"{off.max():.3g} beyond the limit at {np.unravel_index(off.argmax(), off.shape)}"


DECODE = [([1], 1, 1, 64, 16), ([33, 1, 32, 0, 257], 8, 2, 128, 16), ([700, 5], 32, 8, 128, 16), ([64, 63, 65], 12, 4, 96, 12), ([300, 31], 7, 1, 80, 8),
          ([515, 90], 16, 1, 128, 32), ([129, 1024], 40, 2, 64, 64), ([77, 200], 6, 3, 256, 4), ([190, 9], 5, 5, 192, 3), ([45], 3, 1, 17, 1), ([2000, 3], 71, 1, 64, 16)]


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("window", [0, 37])
@pytest.mark.parametrize("contexts,heads,kv_heads,head_dim,page", DECODE)
def test_decode(dtype, window, contexts, heads, kv_heads, head_dim, page):
    b = Batch(len(contexts) * 7 + head_dim, contexts, [1] * len(contexts), heads, kv_heads, head_dim, page, dtype, window)
    b.check(b.decode())


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("head_dim,page", [(128, 16), (64, 12), (192, 16)])
def test_decode_of_long_contexts_in_many_splits(dtype, head_dim, page):
    b = Batch(5, [9001, 1, 4099], [1] * 3, 8, 2, head_dim, page, dtype)
    first = b.decode()
    b.check(first)
    # whatever the hint says, the keys are the sequence's own; and the same call gives the same bits
    b.check(b.decode(max_context=1))
    b.check(b.decode(max_context=2 ** 31 - 1))
    assert np.array_equal(first, b.decode())


def test_decode_of_some_sequences_leaves_the_other_rows():
    b = Batch(11, [40, 50, 60, 70], [1] * 4, 8, 2, 128, 16, "bfloat16")
    got = b.decode(seqs=[3, 1])
    b.check(got, [1, 3])
    assert (got[[0, 2]] == 9.0).all()


PROMPT = [([5, 2], [5, 2], 8, 2, 64, 16), ([40, 300, 7], [9, 33, 2], 8, 2, 128, 16), ([130], [130], 4, 4, 96, 12), ([260, 64], [3, 64], 12, 4, 80, 8),
          ([90, 33], [20, 33], 6, 1, 256, 16), ([50], [50], 5, 5, 192, 3), ([3, 21], [3, 20], 16, 1, 128, 64), ([500, 20], [200, 20], 8, 2, 128, 16),
          ([300], [300], 4, 2, 64, 8), ([1100, 130], [128, 130], 32, 8, 128, 32)]


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("window", [0, 29])
@pytest.mark.parametrize("contexts,queries,heads,kv_heads,head_dim,page", PROMPT)
def test_prompt(dtype, window, contexts, queries, heads, kv_heads, head_dim, page):
    b = Batch(len(contexts) * 13 + head_dim, contexts, queries, heads, kv_heads, head_dim, page, dtype, window)
    b.check(b.prompt(), one_term=True)


# 16-byte aligned rows, run on tcgen05 too: one CTA's row tiles full and not, keys in one, two and four shares, every width of head
LONG = [([130], [130], 4, 4, 128, 16), ([1100, 130], [128, 130], 32, 8, 128, 32), ([700, 64, 3], [40, 64, 3], 8, 1, 64, 12), ([300], [300], 4, 2, 64, 8),
        ([900, 40], [65, 40], 16, 2, 80, 16), ([500, 129], [200, 129], 4, 2, 192, 3), ([400, 2], [129, 2], 6, 3, 136, 64), ([333, 200, 7], [64, 200, 7], 8, 2, 256, 16),
        ([1000], [33], 8, 2, 248, 5), ([260, 257], [256, 257], 3, 3, 40, 16), ([640], [512], 8, 4, 96, 128), ([2100], [130], 12, 4, 64, 16), ([50, 9, 0], [1, 3, 0], 8, 2, 128, 16)]


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("window", [0, 29, 300])
@pytest.mark.parametrize("contexts,queries,heads,kv_heads,head_dim,page", LONG)
@pytest.mark.parametrize("forced", [True, False])
def test_long_portions(monkeypatch, forced, dtype, window, contexts, queries, heads, kv_heads, head_dim, page):
    if forced:          # whatever the number of rows
        monkeypatch.setattr(kv4, "UMMA_MIN_ROWS", 1)
        monkeypatch.setattr(kv4, "UMMA_GROUPS", 0)
    b = Batch(len(contexts) * 17 + head_dim, contexts, queries, heads, kv_heads, head_dim, page, dtype, window, pad=8)
    b.check(b.prompt(), one_term=True, truncated=True)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("window,head_dim", [(0, 64), (16, 128), (0, 192)])
def test_long_portions_with_fewer_keys_than_queries_and_any_hint(monkeypatch, dtype, window, head_dim):
    monkeypatch.setattr(kv4, "UMMA_GROUPS", 0)
    b = Batch(6, [20, 0, 300, 129], [150, 140, 100, 129], 8, 2, head_dim, 16, dtype, window, pad=8)
    for hint in (300, 1, 2 ** 31 - 1):       # how the launch is cut, not what it computes
        b.out.fill_(9.0)
        ops.attention_kv4_prompt(b.qt, b.cache, b.out, *b.args, 4, 150, b.heads, b.scale, hint, b.work, window=window)
        got = b.answer()
        b.check(got, one_term=True, truncated=True)
        assert (got[:130] == 0.0).all() and (got[150:290] == 0.0).all()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("head_dim", [64, 128, 256])
def test_long_portions_leave_the_rows_that_are_not_theirs(monkeypatch, dtype, head_dim):
    monkeypatch.setattr(kv4, "UMMA_GROUPS", 0)
    b = Batch(head_dim, [30, 300, 50], [30, 290, 50], 8, 2, head_dim, 16, dtype, pad=8)
    got = b.prompt(n=2, max_queries=140)
    b.check(got, slice(0, 170), one_term=True, truncated=True)
    assert (got[170:] == 9.0).all()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("head_dim", [64, 128, 192])
def test_a_key_that_is_not_finite_in_a_long_portion(monkeypatch, dtype, head_dim):
    monkeypatch.setattr(kv4, "UMMA_GROUPS", 0)
    b = Batch(head_dim + 1, [500, 160], [200, 160], 8, 2, head_dim, 16, dtype, nan_at=((0, 310),), pad=8)
    got = b.prompt()
    assert np.isnan(got[10:200, :4]).all() and np.isfinite(got[:10]).all() and np.isfinite(got[200:]).all() and np.isfinite(got[:, 4:]).all()
    b.check(got, one_term=True, truncated=True)


def test_prompt_leaves_the_rows_behind_its_sequences():
    b = Batch(3, [30, 300, 50], [30, 200, 1], 8, 2, 128, 16, "bfloat16")
    got = b.prompt(n=2)
    b.check(got, slice(0, 230), one_term=True)
    assert (got[230:] == 9.0).all()


@pytest.mark.parametrize("queries", [20, 200])
def test_a_key_that_is_not_finite_reaches_the_rows_that_see_it_and_no_other(queries):
    b = Batch(4, [queries + 50, 60], [queries, 60], 8, 2, 128, 16, "bfloat16", nan_at=((0, 60),))
    got = b.prompt()
    assert np.isnan(got[11:queries, :4]).all() and np.isfinite(got[:10, :]).all() and np.isfinite(got[queries:]).all() and np.isfinite(got[:, 4:]).all()
    b.check(got, one_term=True)
    d = Batch(4, [400, 61, 60], [1] * 3, 8, 2, 128, 16, "bfloat16", nan_at=((1, 60), (2, 3)))
    got = d.decode()
    assert np.isnan(got[1:, :4]).all() and np.isfinite(got[0]).all() and np.isfinite(got[:, 4:]).all()
    d.check(got)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_hard_softmax(dtype):
    """Queries forty times as loud: one key takes nearly all the weight, and maxima move from tile to tile."""
    b = Batch(9, [3000, 600], [1, 1], 8, 2, 64, 16, dtype, loud=5.0)
    got = b.decode()
    # terms of a score five times as large, so their sums' error too: M 5 * 2^-15 at most, held to M 2^-12
    assert (np.abs(got - b.want) <= b.most * 2.0 ** -12 + np.abs(b.want) * 2.0 ** (-8 if dtype == "bfloat16" else -23)).all()


def test_pages_outside_of_the_cache_are_reported():
    b = Batch(2, [100, 40], [1, 1], 4, 1, 64, 16, "bfloat16")
    tables = b.args[2].clone()
    tables[0, 3] = b.cache.pages
    ops.attention_kv4_decode(b.qt, b.cache, b.out, b.args[0], b.args[1], tables, 4, b.scale, cuda([0, 1]), 2, 100, b.work)
    torch.cuda.synchronize()
    with pytest.raises(TieError, match="page"):
        gemm_select.check_status()
    b.check(b.out.float().cpu().numpy().astype(np.float64).reshape(b.want.shape), [1])       # the other sequence is right
    ops.attention_kv4_decode(b.qt, b.cache, b.out, b.args[0], b.args[1], b.args[2][:, :2].contiguous(), 4, b.scale, cuda([1, 0]), 2, 100, b.work)
    torch.cuda.synchronize()
    with pytest.raises(TieError, match="too short"):
        gemm_select.check_status()


def test_other_streams_and_graphs():
    b = Batch(8, [1500, 700], [1, 1], 8, 2, 128, 16, "bfloat16")
    want = b.decode()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        b.out.fill_(0.0)
        ops.attention_kv4_decode(b.qt, b.cache, b.out, *b.args, b.heads, b.scale, cuda([0, 1]), 2, 1500, b.work)
    side.synchronize()
    assert np.array_equal(want, b.answer())
    seqs = cuda([0, 1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.attention_kv4_decode(b.qt, b.cache, b.out, *b.args, b.heads, b.scale, seqs, 2, 1500, b.work)
    b.out.fill_(0.0)
    graph.replay()
    assert np.array_equal(want, b.answer())


@pytest.mark.parametrize("dtype,head_dim,contexts", [("bfloat16", 64, [3000]), ("bfloat16", 128, [700, 300]), ("bfloat16", 256, [3000]), ("float32", 128, [2500])])
def test_long_portions_on_other_streams_and_in_graphs(monkeypatch, dtype, head_dim, contexts):
    """With the keys in one share and in several; queries and contexts that change between replays are the ones that count."""
    monkeypatch.setattr(kv4, "UMMA_GROUPS", 0)
    b = Batch(41, contexts, [130] * len(contexts), 4, 2, head_dim, 16, dtype, pad=8)
    want = b.prompt()
    b.check(want, one_term=True, truncated=True)
    args = len(contexts), 130, b.heads, b.scale, max(contexts), b.work
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b.out.fill_(0.0)
        ops.attention_kv4_prompt(b.qt, b.cache, b.out, *b.args, *args)
    side.synchronize()
    assert np.array_equal(want, b.answer())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.attention_kv4_prompt(b.qt, b.cache, b.out, *b.args, *args)
    b.args[1].sub_(140)         # fewer keys: every row sees other ones
    graph.replay()
    fewer = b.answer()
    ops.attention_kv4_prompt(b.qt, b.cache, b.out, *b.args, *args)
    assert np.array_equal(fewer, b.answer()) and not np.array_equal(fewer, want)
    b.args[1].add_(140)
    b.out.fill_(0.0)
    graph.replay()
    assert np.array_equal(want, b.answer())


def test_calls_at_the_same_time_with_workspaces_of_their_own():
    batches = [Batch(20 + i, [4000, 300, 2500], [1] * 3, 8, 2, 128, 16, "bfloat16") for i in range(2)]
    want = [b.decode() for b in batches]
    streams, seqs = [torch.cuda.Stream() for _ in batches], cuda([0, 1, 2])
    torch.cuda.synchronize()
    for _ in range(20):
        for b, stream in zip(batches, streams):
            with torch.cuda.stream(stream):
                b.out.fill_(9.0)
                ops.attention_kv4_decode(b.qt, b.cache, b.out, *b.args, b.heads, b.scale, seqs, 3, 4000, b.work)
    for b, w in zip(batches, want):
        assert np.array_equal(b.answer(), w)


def test_a_sequence_that_is_listed_twice():
    b = Batch(31, [5000, 70], [1, 1], 8, 2, 128, 16, "bfloat16")
    b.check(b.decode(seqs=[0, 1, 0]))


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("T,heads,kv_heads,head_dim,rot", [(1, 4, 2, 64, 64), (7, 8, 8, 128, 128), (300, 6, 2, 128, 128), (2050, 2, 1, 64, 64), (5, 3, 1, 48, 32), (260, 4, 2, 256, 0)])
def test_queries_and_keys_prepared_in_place(dtype, T, heads, kv_heads, head_dim, rot):
    """One launch over both does, bit for bit, what one over the queries and one over the keys do; values stay."""
    rng = np.random.default_rng(T + head_dim)
    width = (heads + 2 * kv_heads) * head_dim
    x = cuda(rng.standard_normal((T, width)), DT[dtype])
    qw, kw = (cuda(rng.random(head_dim) + 0.5, torch.float32) for _ in range(2))
    table = cuda(10000.0 ** (-np.arange(0, rot, 2) / rot), torch.float32) if rot else None
    pos = cuda(rng.integers(0, 40000, T))
    want = x.clone()
    q, k = want[:, :heads * head_dim], want[:, heads * head_dim:(heads + kv_heads) * head_dim]
    ops.qk_norm_rope_append(q, qw, None, 1e-6, 0.0, table, pos, None, None, None, heads, kv_heads, head_dim, write_kv=False)
    ops.qk_norm_rope_append(k, kw, None, 1e-5, 0.0, table, pos, None, None, None, kv_heads, kv_heads, head_dim, write_kv=False)
    ops.qk_norm_rope(x, qw, kw, 1e-6, 1e-5, table, pos, heads, kv_heads, head_dim)
    assert torch.equal(x, want)


@pytest.mark.parametrize("T,heads,kv_heads,head_dim", [(1, 4, 2, 64), (9, 6, 2, 128), (3, 3, 1, 48)])
def test_queries_and_keys_out_of_partial_sums(T, heads, kv_heads, head_dim):
    """What goes back in place is what `qk_norm_rope_append` puts into a bfloat16 cache."""
    rng = np.random.default_rng(T)
    width = (heads + 2 * kv_heads) * head_dim
    sums = ops.SplitSum(cuda(rng.standard_normal((3, T, width)), torch.float32).reshape(-1), 3, T, width)
    qw, kw = (cuda(rng.random(head_dim) + 0.5, torch.float32) for _ in range(2))
    table = cuda(10000.0 ** (-np.arange(0, head_dim, 2) / head_dim), torch.float32)
    pos, slots = cuda(rng.integers(0, 40000, T)), cuda(np.arange(T))
    got, want = (torch.zeros(T, width, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    planes = [torch.zeros(1, kv_heads, 16, head_dim, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    ops.qk_norm_rope_append(want, qw, kw, 1e-6, 1e-5, table, pos, slots, *planes, heads, kv_heads, head_dim, partial=sums)
    ops.qk_norm_rope(got, qw, kw, 1e-6, 1e-5, table, pos, heads, kv_heads, head_dim, partial=sums)
    for i, plane in enumerate(planes):
        at = (heads + i * kv_heads) * head_dim
        want[:, at:at + kv_heads * head_dim] = plane[0, :, :T].transpose(0, 1).reshape(T, -1)
    assert torch.equal(got, want) and bool((got != 0).any(0).all())


# ---- step tables

def device_tables(requests, columns, pages):
    return dict(lens=cuda(np.zeros(requests)), tables=cuda(np.zeros((requests, columns))), free_pages=cuda(np.arange(pages - 1, -1, -1)), free_count=cuda([pages]))


def same(arrays, want):
    torch.cuda.synchronize()
    for name, w in want.items():
        assert np.array_equal(getattr(arrays, name).cpu().numpy(), w), name


@pytest.mark.parametrize("page,requests,seqs,pages", [(16, 9, 5, 400), (1, 40, 17, 4000), (12, 700, 600, 9000), (48, 3000, 2000, 6000)])
def test_step_tables_follow_the_cache_manager(page, requests, seqs, pages):
    """Steps of random requests and counts, with requests released in between: every array as the host's cache manager has it."""
    rng = np.random.default_rng(page + seqs)
    columns = 64
    state, host = device_tables(requests, columns, pages), plain.HostTables(pages, page)
    for step in range(8):
        who = rng.permutation(requests)[:seqs].astype(np.int32)
        who[rng.random(seqs) < 0.1] = -1
        counts = rng.integers(0, 3 + page // 4, seqs).astype(np.int32)
        counts = np.where(who >= 0, np.minimum(counts, [columns * page // 8] * seqs), 1).astype(np.int32)
        rows = int(counts.sum()) + int(rng.integers(0, 5))
        arrays = ops.step_arrays(seqs, rows, columns)
        if step % 3 == 2:                    # planned first, without a commit: the same arrays, and the state stays
            before = {k: v.clone() for k, v in state.items() if k != "tables"}
            ops.step_tables(cuda(who), cuda(counts), **state, page_size=page, arrays=arrays, commit=False)
            assert all(torch.equal(state[k], v) for k, v in before.items())
            arrays = ops.StepArrays(*(torch.full_like(t, -9) for t in arrays))
        ops.step_tables(cuda(who), cuda(counts), **state, page_size=page, arrays=arrays)
        same(arrays, host.step(who.tolist(), counts.tolist(), rows, columns))
        assert int(state["free_count"]) == host.manager.num_free()
        if step % 2:
            gone = rng.permutation(requests)[:requests // 3].astype(np.int32)
            gone[::5] = -1
            status = cuda([7])
            ops.release_tables(cuda(gone), **state, page_size=page, status=status)
            host.release(gone.tolist())
            assert int(status) == 0 and int(state["free_count"]) == host.manager.num_free()
        lens = np.zeros(requests, np.int32)
        for r, length in host.lens.items():
            lens[r] = length
        assert np.array_equal(state["lens"].cpu().numpy(), lens)


@pytest.mark.parametrize("case,bits", [("pages", ops.TABLES_NO_PAGES), ("short", ops.TABLES_SHORT), ("rows", ops.TABLES_ROWS), ("outside", ops.TABLES_BAD_REQUEST),
                                       ("negative", ops.TABLES_BAD_REQUEST), ("twice", ops.TABLES_BAD_REQUEST), ("length", ops.TABLES_BAD_REQUEST),
                                       ("count", ops.TABLES_BAD_REQUEST)])
def test_step_tables_refuse_a_step_whole(case, bits):
    state = device_tables(6, 4, 7)
    ops.step_tables(cuda([2, 4]), cuda([9, 3]), **state, page_size=4, arrays=ops.step_arrays(2, 16, 4))
    who, counts, rows = [2, 0, 5], [1, 5, 4], 12
    if case == "pages":
        counts = [1, 9, 7]
        rows = 20
    elif case == "short":
        counts = [8, 1, 1]
    elif case == "rows":
        rows = 9
    elif case == "outside":
        who = [2, 6, 5]
    elif case == "negative":
        who = [2, -2, 5]
    elif case == "twice":
        who = [2, 5, 5]
    elif case == "length":
        state["lens"][0] = -1
    else:
        counts = [1, -1, 4]
    before = {k: v.clone() for k, v in state.items()}
    arrays = ops.step_arrays(3, rows, 4)
    ops.step_tables(cuda(who), cuda(counts), **state, page_size=4, arrays=arrays)
    same(arrays, dict(query_start=np.zeros(4), context_lens=np.zeros(3), positions=np.zeros(rows), seq_of_row=np.full(rows, -1), slots=np.full(rows, -1),
                      block_tables=np.zeros((3, 4)), free_left=[3], status=[bits]))
    assert all(torch.equal(state[k], v) for k, v in before.items())


def test_release_refuses_whole():
    state = device_tables(3, 4, 5)
    ops.step_tables(cuda([0, 2]), cuda([5, 3]), **state, page_size=4, arrays=ops.step_arrays(2, 8, 4))
    before = {k: v.clone() for k, v in state.items()}
    status = cuda([0])
    for who in ([0, 0], [3], [-2]):
        ops.release_tables(cuda(who), **state, page_size=4, status=status)
        assert int(status) == ops.TABLES_BAD_REQUEST and all(torch.equal(state[k], v) for k, v in before.items())


def test_step_tables_of_no_sequences_and_of_no_rows():
    state = device_tables(3, 4, 5)
    arrays = ops.step_arrays(0, 3, 4)
    ops.step_tables(cuda([]), cuda([]), **state, page_size=4, arrays=arrays)
    same(arrays, dict(query_start=[0], slots=[-1] * 3, positions=[0] * 3, seq_of_row=[-1] * 3, free_left=[5], status=[0]))
    arrays = ops.step_arrays(2, 0, 4)
    ops.step_tables(cuda([1, -1]), cuda([0, 0]), **state, page_size=4, arrays=arrays)
    same(arrays, dict(query_start=[0] * 3, context_lens=[0, 0], block_tables=np.zeros((2, 4)), status=[0]))


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_a_run_of_steps_as_they_would_be_used(dtype):
    """Three requests: portions of prompts, then tokens one by one, in one captured step that the GPU's own lengths move on: tables, append and
    attention together, against attention over everything appended so far."""
    heads, kv_heads, dim, page, pages = 8, 2, 128, 16, 40
    rng = np.random.default_rng(0)
    state, cache, work = device_tables(5, 12, pages), ops.kv4_cache(pages, kv_heads, page, dim), ops.kv4_workspace(heads, kv_heads, dim)
    who = cuda([4, 1, 2])
    said = {i: [] for i in range(3)}
    graph, fixed = None, None
    for step, counts in enumerate([[70, 5, 33], [40, 2, 3]] + [[1, 1, 1]] * 6):
        T = sum(counts)
        qkv = rounded(rng.standard_normal((T, (heads + 2 * kv_heads) * dim)), dtype)
        rows = cuda(qkv, DT[dtype])

        def run(rows, counts_t, arrays, out):
            ops.step_tables(who, counts_t, **state, page_size=page, arrays=arrays)
            q, k, v = rows.split([heads * dim, kv_heads * dim, kv_heads * dim], 1)
            ops.kv4_append(k, v, arrays.slots, cache)
            if T > 3:
                ops.attention_kv4_prompt(q, cache, out, arrays.query_start, arrays.context_lens, arrays.block_tables, 3, max(counts), heads, dim ** -0.5, 192, work)
            else:
                ops.attention_kv4_decode(q, cache, out, arrays.query_start, arrays.context_lens, arrays.block_tables, heads, dim ** -0.5, seqs, 3, 192, work)
        seqs = cuda([0, 1, 2])
        if T > 3 or step == 2:
            out, arrays = torch.empty(T, heads * dim, dtype=DT[dtype], device="cuda"), ops.step_arrays(3, T, 12)
            run(rows, cuda(counts), arrays, out)
        elif graph is None:
            fixed = (rows.clone(), cuda(counts), ops.step_arrays(3, 3, 12), torch.empty(3, heads * dim, dtype=DT[dtype], device="cuda"), seqs)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                run(*fixed[:4])
            graph.replay()
            out, arrays = fixed[3], fixed[2]
        else:
            fixed[0].copy_(rows)
            graph.replay()
        torch.cuda.synchronize()
        gemm_select.check_status()
        assert int(arrays.status) == 0
        got, row = out.float().cpu().numpy().astype(np.float64).reshape(T, heads, dim), 0
        for i, c in enumerate(counts):
            part = qkv[row:row + c].reshape(c, heads + 2 * kv_heads, dim)
            said[i].append(part)
            seen = np.concatenate(said[i])
            (kc, kw), (vc, vw) = plain.quantise(seen[:, heads:heads + kv_heads], seen[:, heads + kv_heads:])
            kx, vx = plain.values(kc, kw, dim), plain.values(vc, vw, dim)
            for h in range(heads):
                want = plain.attention(part[:, h].astype(np.float64), kx[:, h // 4], vx[:, h // 4], np.arange(len(seen) - c, len(seen)), dim ** -0.5)
                limit = np.abs(vx[:, h // 4]).max() * (2.0 ** -15 if dtype == "float32" else 2.0 ** -14 + 2.0 ** -8) + np.abs(want) * 2.0 ** (-23 if dtype == "float32" else -8)
                assert (np.abs(got[row:row + c, h] - want) <= limit * 1.001).all(), (step, i, h)
            row += c
    assert state["lens"].tolist() == [0, 13, 42, 0, 116]
