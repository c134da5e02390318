"""Attention over a cache in 4 bits where there is little to read: sequences and rows without keys, tables that are no wider than they have to
be, portions that bring more tokens than a call takes. Tolerances: test_kv4_gpu.py."""
import numpy as np
import pytest
import torch

from test_kv4_gpu import DT, PROMPT, Batch, cuda
from tiny_inference_engine_b200 import ops
from tiny_inference_engine_b200.errors import TieError
from tiny_inference_engine_b200.ops import gemm_select, kv4

pytestmark = pytest.mark.gpu


def narrow(b, page, columns=None):
    """The batch's tables as wide as its longest context needs (or `columns`), with -1 in every entry that holds no page and behind the last row."""
    n = len(b.contexts)
    pages = [-(-c // page) for c in b.contexts]
    width = max(pages) if columns is None else columns
    room = np.full(n * width + 64, -1, np.int32)
    rows = room[:n * width].reshape(n, width)
    old = b.args[2].cpu().numpy()
    for i, p in enumerate(pages):
        rows[i, :min(p, width)] = old[i, :min(p, width)]
    b.room = cuda(room)
    b.args = (b.args[0], b.args[1], b.room[:n * width].view(n, width))
    return b


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("window", [0, 37])
@pytest.mark.parametrize("contexts,heads,kv_heads,head_dim,page", [([17, 0, 30, 0], 8, 2, 128, 16), ([0, 5, 0], 4, 4, 64, 8), ([1, 0], 71, 1, 64, 1), ([0, 200, 0], 32, 2, 192, 64),
                                                                  ([3000, 0, 40, 0], 6, 1, 256, 16)])
def test_tokens_of_sequences_without_keys(dtype, window, contexts, heads, kv_heads, head_dim, page):
    b = narrow(Batch(len(contexts) + head_dim, contexts, [1] * len(contexts), heads, kv_heads, head_dim, page, dtype, window), page)
    for hint in (max(contexts), 1, 2 ** 31 - 1):
        b.out.fill_(9.0)
        got = b.decode(max_context=hint)           # (looks at the status too: no entry that is no page is asked for)
        b.check(got)
        assert (got[[i for i, c in enumerate(contexts) if c == 0]] == 0.0).all()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("window", [0, 16])
@pytest.mark.parametrize("heads,kv_heads,head_dim,page", [(8, 2, 128, 16), (3, 3, 64, 8), (4, 1, 256, 4), (6, 2, 192, 1)])
def test_short_portions_with_fewer_keys_than_queries(dtype, window, heads, kv_heads, head_dim, page):
    b = narrow(Batch(head_dim, [20, 0, 5, 33], [40, 9, 21, 33], heads, kv_heads, head_dim, page, dtype, window), page)
    got = b.prompt()
    b.check(got, one_term=True)
    assert (got[:20] == 0.0).all() and (got[40:49] == 0.0).all() and (got[49:65] == 0.0).all()


@pytest.mark.parametrize("columns", [0, 2])
@pytest.mark.parametrize("window", [0, 64])
def test_tables_that_are_too_short_are_reported_and_not_read_behind(columns, window):
    b = narrow(Batch(12, [900, 0, 30], [1] * 3, 8, 2, 64, 16, "bfloat16", window), 16, columns)
    seqs = cuda([0, 1, 2])
    ops.attention_kv4_decode(b.qt, b.cache, b.out, *b.args, b.heads, b.scale, seqs, 3, 900, b.work, window=window)
    torch.cuda.synchronize()
    with pytest.raises(TieError, match="too short"):
        gemm_select.check_status()
    got = b.out.float().cpu().numpy().astype(np.float64).reshape(b.want.shape)
    b.check(got, [1, 2] if columns else [1])
    # sequences without keys need no columns at all
    ops.attention_kv4_decode(b.qt, b.cache, b.out, *b.args, b.heads, b.scale, cuda([1]), 1, 900, b.work, window=window)
    assert (b.answer()[1] == 0.0).all()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("heads,kv_heads", [(2, 2), (6, 2), (8, 2), (7, 1)])
@pytest.mark.parametrize("most", [1, 3, 5])
def test_short_portions_of_more_tokens_than_the_call_takes(dtype, heads, kv_heads, most):
    """The last block of rows ends inside of a token's neighbours: those are not touched. Every count of rows a CTA (4, 8, 16) and of heads a group."""
    contexts, queries = [30, 300, 50, 7], [8, 40, 2, 7]
    b = Batch(most + heads, contexts, queries, heads, kv_heads, 64, 16, dtype)
    got = b.prompt(max_queries=most)
    taken = np.concatenate([b.start[i] + np.arange(min(q, most)) for i, q in enumerate(queries)])
    b.check(got, taken, one_term=True)
    rest = np.setdiff1d(np.arange(sum(queries)), taken)
    assert len(rest) and (got[rest] == 9.0).all()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("heads,kv_heads", [(2, 2), (6, 2), (16, 2)])
def test_tokens_of_listed_sequences_that_bring_several(dtype, heads, kv_heads):
    """A listed sequence's first row, wherever it sits, and no other."""
    b = Batch(heads, [40, 2000, 3], [3, 9, 1], heads, kv_heads, 128, 16, dtype)
    got = b.decode(seqs=[1, 2, 0])
    b.check(got, [0, 3, 12])
    assert (np.delete(got, [0, 3, 12], 0) == 9.0).all()


@pytest.mark.parametrize("window", [0, 29])
@pytest.mark.parametrize("contexts,queries,heads,kv_heads,head_dim,page", PROMPT)
def test_short_portions_have_weights_of_two_terms(window, contexts, queries, heads, kv_heads, head_dim, page):
    """Rows that are not 16-byte aligned stay with the kernel of few rows, whatever their number: weights enter with 16 bits."""
    b = Batch(len(contexts) * 13 + head_dim, contexts, queries, heads, kv_heads, head_dim, page, "bfloat16", window)
    assert b.qt.stride(0) % 8
    b.check(b.prompt(), one_term=False)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_planes_of_more_than_4_gb(monkeypatch, dtype):
    """A sequence's pages at the far end of the planes give the bits that they give at the near one: append, read, tokens and both kinds of portions."""
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("planes of 10 GB")
    kv_heads, heads, dim, page, n = 2, 8, 256, 64, 300
    pages = (1 << 32) // (kv_heads * page * dim // 2) + 8              # a plane of codes: 2^32 bytes and 8 pages more
    big, small = ops.kv4_cache(pages, kv_heads, page, dim), ops.kv4_cache(5, kv_heads, page, dim)
    assert big.k_codes.numel() > 1 << 32
    rng = np.random.default_rng(3)
    k, v = (cuda(rng.standard_normal((n, kv_heads * dim)), DT[dtype]) for _ in range(2))
    q = cuda(rng.standard_normal((n, heads * dim)), DT[dtype])
    work = ops.kv4_workspace(heads, kv_heads, dim)
    got = []
    for cache, first in ((small, 0), (big, pages - 5)):
        table = first + np.array([[3, 1, 0, 4, 2]])
        at = np.arange(n)
        slots = cuda(table[0, at // page] * page + at % page)
        assert int(slots.max()) < 2 ** 31
        ops.kv4_append(k, v, slots, cache)
        out = [torch.empty_like(x) for x in (k, v, q, q, q)]
        ops.kv4_read(cache, slots, out[0], out[1])
        for i, min_groups, rows in ((2, 1 << 30, n), (3, 0, n), (4, 0, 1)):
            monkeypatch.setattr(kv4, "UMMA_GROUPS", min_groups), monkeypatch.setattr(kv4, "UMMA_FEW_GROUPS", min_groups)
            out[i].zero_()
            args = q, cache, out[i], cuda([0, rows]), cuda([n]), cuda(table)
            if rows == 1:
                ops.attention_kv4_decode(*args, heads, dim ** -0.5, cuda([0]), 1, n, work)
            else:
                ops.attention_kv4_prompt(*args, 1, n, heads, dim ** -0.5, n, work)
        torch.cuda.synchronize()
        gemm_select.check_status()
        got.append(out)
    assert all(torch.equal(x, y) for x, y in zip(*got)) and bool((got[0][3] != 0).any(1).all())


def test_step_tables_of_the_most_sequences_and_requests_and_of_more():
    from tiny_inference_engine_b200.errors import InvalidArgument
    n, held = 8192, 1 << 17
    state = dict(lens=cuda(np.zeros(held)), tables=cuda(np.zeros((held, 2))), free_pages=cuda(np.arange(2 * n)), free_count=cuda([2 * n]))
    who = np.random.default_rng(0).permutation(held)[:n]
    arrays = ops.step_arrays(n, 3 * n, 2)
    ops.step_tables(cuda(who), cuda(np.full(n, 3)), **state, page_size=2, arrays=arrays)
    assert int(arrays.status) == 0 and int(arrays.free_left) == 0 and int(state["free_count"]) == 0
    assert np.array_equal(state["lens"].cpu().numpy()[who], np.full(n, 3)) and int(state["lens"].sum()) == 3 * n
    # pages come off the end of the stack, in the order of the sequences
    assert np.array_equal(arrays.block_tables.cpu().numpy().reshape(-1), np.arange(2 * n)[::-1])
    pages = arrays.block_tables.cpu().numpy()
    assert np.array_equal(arrays.slots.cpu().numpy().reshape(n, 3), np.stack([pages[:, 0] * 2, pages[:, 0] * 2 + 1, pages[:, 1] * 2], 1))
    status = cuda([7])
    ops.release_tables(cuda(who), **state, page_size=2, status=status)
    assert int(status) == 0 and int(state["free_count"]) == 2 * n and int(state["lens"].abs().sum()) == 0
    assert np.array_equal(state["free_pages"].cpu().numpy(), np.arange(2 * n)[::-1])
    with pytest.raises(InvalidArgument, match="8193 sequences"):
        ops.step_tables(cuda(np.full(n + 1, -1)), cuda(np.zeros(n + 1)), **state, page_size=2, arrays=ops.step_arrays(n + 1, 4, 2))
    with pytest.raises(InvalidArgument, match="8193 sequences"):
        ops.release_tables(cuda(np.full(n + 1, -1)), **state, page_size=2, status=status)
    state["lens"], state["tables"] = cuda(np.zeros(held + 1)), cuda(np.zeros((held + 1, 2)))
    with pytest.raises(InvalidArgument, match="131073 requests"):
        ops.step_tables(cuda([0]), cuda([1]), **state, page_size=2, arrays=ops.step_arrays(1, 4, 2))


def test_entries_of_a_list_that_name_no_sequence_are_left_out():
    b = Batch(19, [40, 900], [1, 1], 8, 2, 64, 16, "bfloat16")
    got = b.decode(seqs=[-1, 1, 2, 2 ** 31 - 1])
    b.check(got, [1])
    assert (got[0] == 9.0).all()


def test_calls_of_two_graphs_that_run_at_the_same_time():
    """Each with a workspace of its own, replayed in two streams; and one after the other with one workspace."""
    a, b = (Batch(50 + i, [4000, 300], [1, 1], 8, 2, 128, 16, "bfloat16") for i in range(2))
    want = [a.decode(), b.decode()]
    seqs, graphs = cuda([0, 1]), []
    for x, work in ((a, a.work), (b, b.work), (b, a.work)):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            x.out.fill_(9.0)
            ops.attention_kv4_decode(x.qt, x.cache, x.out, *x.args, x.heads, x.scale, seqs, 2, 4000, work)
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    for x, w in zip((a, b), want):
        assert np.array_equal(x.answer(), w)
    for _ in range(5):
        graphs[0].replay(), graphs[2].replay()
    for x, w in zip((a, b), want):
        assert np.array_equal(x.answer(), w)
