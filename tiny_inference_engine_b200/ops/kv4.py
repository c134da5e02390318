"""A key/value cache in 4 bits whose step tables are built on the GPU: Python faces of csrc/kv4_cache.cu, csrc/attention_kv4.cu,
csrc/attention_prompt_kv4.cu and csrc/step_tables.cu (checks of the arguments, then one or two launches on the current stream).

A token's key (and value) of one kv head is `head_dim` numbers, padded with zeros to whole 64s, in groups of 32. Of a group, with
lo = min(0, its least) and hi = max(0, its largest):

    s = (hi - lo) / 15 in 32 bits, at least 2^-100, rounded up to three significant bits
    z = round(-lo / s),   code = clamp(round(x / s) + z, 0, 15)     (ties to even),   what it stands for: s (code - z)

so that every value is a bfloat16 number within s of what was appended, and costs 4.5 bits. Codes lie in padded / 2 bytes, dimension d in
byte d // 2, the even one in the low bits; a group's 16-bit word holds s as bfloat16 (its low five bits are zero) and z in its low four. A token
and head whose key or value holds a number that is not finite, or one of magnitude 2^120 or more, gets the key words 0x7fc0, zero
value words and zero codes: rows that see that key are NaN, no other is.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from ..errors import InvalidArgument
from .library import call, library


class Kv4Cache(NamedTuple):
    """The planes of one layer: codes uint8 [pages, kv_heads, page_size, padded / 2], words int16 [pages, kv_heads, page_size, padded / 32]
    of keys and of values; padded is head_dim rounded up to whole 64s."""
    k_codes: torch.Tensor
    k_words: torch.Tensor
    v_codes: torch.Tensor
    v_words: torch.Tensor
    head_dim: int

    @property
    def pages(self) -> int:
        return self.k_codes.shape[0]

    @property
    def kv_heads(self) -> int:
        return self.k_codes.shape[1]

    @property
    def page_size(self) -> int:
        return self.k_codes.shape[2]


class Kv4Workspace(NamedTuple):
    """Where the splits of a row's keys leave their sums. Calls that run one after the other may share it (`counters` is zero between them);
    calls that may run at the same time, in two streams or two captured graphs, need one each."""
    scratch: torch.Tensor       # float32
    counters: torch.Tensor      # int32, zeros


class StepArrays(NamedTuple):
    """The index arrays of a step of n sequences in room for `rows` rows, all int32: what `step_tables` writes."""
    query_start: torch.Tensor       # [n + 1]
    context_lens: torch.Tensor      # [n] length after the step
    positions: torch.Tensor         # [rows]
    seq_of_row: torch.Tensor        # [rows]; -1 behind the last sequence
    slots: torch.Tensor             # [rows]; -1 behind the last sequence and in rows of padding
    block_tables: torch.Tensor      # [n, columns]; zeros behind a sequence's pages
    free_left: torch.Tensor         # [1] pages that the step leaves free
    status: torch.Tensor            # [1] 0, or the TABLES_* bits of what made the step impossible


TABLES_NO_PAGES, TABLES_SHORT, TABLES_ROWS, TABLES_BAD_REQUEST = 1, 2, 4, 8


def _need(cond, msg: str) -> None:
    if not cond:
        raise InvalidArgument(msg)


def _one_device(what: str, *ts) -> None:
    for t in ts:
        if t is not None and not t.is_cuda:
            raise InvalidArgument("kernel arguments must be CUDA tensors: the engine has no CPU path")
    devices = {t.device for t in ts if t is not None}
    _need(len(devices) == 1 and next(iter(devices)).index == torch.cuda.current_device(),
          f"{what}: all tensors must be on the current device, got {sorted(map(str, devices))}")


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _int32(what: str, name: str, t, *shape) -> None:
    _need(t.dtype == torch.int32 and t.is_contiguous() and tuple(t.shape) == shape, f"{what}: {name} must be contiguous int32 {list(shape)}")


def _float_code(what: str, *ts) -> int:
    codes = {torch.float32: 0, torch.bfloat16: 1}
    _need(ts[0].dtype in codes and all(t.dtype == ts[0].dtype for t in ts), f"{what}: rows must be float32 or bfloat16, all alike")
    return codes[ts[0].dtype]


def kv4_cache(pages: int, kv_heads: int, page_size: int, head_dim: int, device="cuda") -> Kv4Cache:
    """An empty cache for one layer (of any number of requests)."""
    _need(pages > 0 and kv_heads > 0 and page_size > 0 and 0 < head_dim <= 256 and pages * page_size < 2 ** 31,
          f"kv4_cache: bad sizes (pages {pages}, kv heads {kv_heads}, page size {page_size}, head size {head_dim}, at most 256)")
    padded = -(-head_dim // 64) * 64

    def plane(width, dtype):
        return torch.zeros(pages, kv_heads, page_size, width, dtype=dtype, device=device)
    return Kv4Cache(plane(padded // 2, torch.uint8), plane(padded // 32, torch.int16), plane(padded // 2, torch.uint8), plane(padded // 32, torch.int16), head_dim)


def _check_cache(what: str, c: Kv4Cache) -> None:
    _need(0 < c.head_dim <= 256, f"{what}: head size {c.head_dim} is not in 1..256")
    padded = -(-c.head_dim // 64) * 64
    for codes, words in ((c.k_codes, c.k_words), (c.v_codes, c.v_words)):
        _need(codes.dim() == 4 and codes.dtype == torch.uint8 and codes.shape[3] == padded // 2 and words.dtype == torch.int16 and
              tuple(words.shape) == (*codes.shape[:3], padded // 32) and codes.shape == c.k_codes.shape and codes.is_contiguous() and words.is_contiguous(),
              f"{what}: planes must be contiguous, codes uint8 [pages, kv_heads, page_size, {padded // 2}] and words int16 [..., {padded // 32}]")
        _need(codes.data_ptr() % 16 == 0 and words.data_ptr() % 16 == 0, f"{what}: planes must be 16-byte aligned")
    _need(c.pages > 0 and c.kv_heads > 0 and c.page_size > 0 and c.pages * c.page_size < 2 ** 31, f"{what}: slots must be 32-bit numbers, of one page at least")


def _check_rows(what: str, c: Kv4Cache, k, v, slots) -> int:
    _check_cache(what, c)
    dtype = _float_code(what, k, v)
    _need(k.dim() == 2 and k.shape == v.shape and k.shape[1] == c.kv_heads * c.head_dim and all(t.stride(1) == 1 or t.shape[1] == 1 for t in (k, v)),
          f"{what}: k and v must be [T, {c.kv_heads * c.head_dim}] with contiguous rows")
    _int32(what, "slots", slots, k.shape[0])
    _one_device(what, k, v, slots, *c[:4])
    return dtype


def kv4_append(k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, cache: Kv4Cache) -> None:
    """k, v [T, kv_heads * head_dim] (float32 or bfloat16, rows may be strided) into the cache at slots[t]; slot < 0 writes nothing. The slots of a
    call must differ: of a slot that is named twice it is not said which row it keeps, or which part of either. A slot outside of the cache
    writes nothing either and is reported by `gemm_select.check_status`."""
    dtype = _check_rows("kv4_append", cache, k, v, slots)
    call("tie_kv4_append", dtype, k.data_ptr(), v.data_ptr(), k.stride(0), v.stride(0), slots.data_ptr(), cache.k_codes.data_ptr(),
         cache.k_words.data_ptr(), cache.v_codes.data_ptr(), cache.v_words.data_ptr(), k.shape[0], cache.kv_heads, cache.head_dim, cache.page_size,
         cache.pages, _stream())


def kv4_read(cache: Kv4Cache, slots: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> None:
    """The values that the cache holds at slots[t] into k, v [T, kv_heads * head_dim] (float32 or bfloat16, exact in both); rows whose slot is below
    zero are left as they are."""
    dtype = _check_rows("kv4_read", cache, k, v, slots)
    call("tie_kv4_read", dtype, cache.k_codes.data_ptr(), cache.k_words.data_ptr(), cache.v_codes.data_ptr(), cache.v_words.data_ptr(), slots.data_ptr(),
         k.data_ptr(), v.data_ptr(), k.stride(0), v.stride(0), k.shape[0], cache.kv_heads, cache.head_dim, cache.page_size, cache.pages, _stream())


def kv4_workspace(q_heads: int, kv_heads: int, head_dim: int, device="cuda") -> Kv4Workspace:
    """The workspace of `attention_kv4_decode` and `attention_kv4_prompt` for heads of these sizes, whatever the batch."""
    _need(q_heads > 0 and kv_heads > 0 and q_heads % kv_heads == 0 and 0 < head_dim <= 256, "kv4_workspace: bad sizes")
    ctas = library().tie_attention_kv4_ctas()
    return Kv4Workspace(torch.empty(ctas * 16 * (head_dim + 2), dtype=torch.float32, device=device), torch.zeros(ctas, dtype=torch.int32, device=device))


def _check_attention(what, q, cache, out, query_start, context_lens, block_tables, q_heads, workspace, window, n: int, scale,
                     max_context, max_queries: int, seq_list=None) -> int:
    _check_cache(what, cache)
    dtype = _float_code(what, q, out)
    _need(q_heads > 0 and q_heads % cache.kv_heads == 0, f"{what}: {q_heads} heads are not a multiple of {cache.kv_heads} kv heads")
    width = q_heads * cache.head_dim
    _need(q.dim() == 2 and q.shape[1] >= width and (q.stride(1) == 1 or q.shape[1] == 1), f"{what}: q must be [T, {width}] or wider, with contiguous rows")
    _need(tuple(out.shape) == (q.shape[0], width) and out.is_contiguous(), f"{what}: out must be contiguous [T, {width}]")
    S = context_lens.numel()
    _int32(what, "query_start", query_start, S + 1)
    _int32(what, "context_lens", context_lens, S)
    _need(block_tables.dim() == 2, f"{what}: block_tables must be [sequences, pages]")
    _int32(what, "block_tables", block_tables, S, block_tables.shape[1])
    _need(0 <= n <= S or seq_list is not None, f"{what}: {n} of {S} sequences")
    _need(0 <= n <= 65535, f"{what}: at most 65,535 sequences a call, got {n}")
    _need(0 <= window < 2 ** 30, f"{what}: bad window {window}")
    ctas = library().tie_attention_kv4_ctas()
    _need(workspace.scratch.dtype == torch.float32 and workspace.scratch.is_contiguous() and workspace.scratch.numel() >= ctas * 16 * (cache.head_dim + 2) and
          workspace.counters.dtype == torch.int32 and workspace.counters.is_contiguous() and workspace.counters.numel() >= ctas,
          f"{what}: the workspace is too small (kv4_workspace makes one)")
    _need(scale > 0 and max_context >= 0 and 0 <= max_queries < 2 ** 30, f"{what}: the scale must be positive, max_context and max_queries not negative")
    _need(seq_list is None or (seq_list.dtype == torch.int32 and seq_list.dim() == 1 and seq_list.is_contiguous() and seq_list.numel() >= n),
          f"{what}: seq_list must be int32 [n_list]")
    _one_device(what, q, out, query_start, context_lens, block_tables, seq_list, *workspace, *cache[:4])
    return dtype


def _rows_kernel(dtype, q, cache, out, query_start, context_lens, block_tables, max_queries, q_heads, scale, window, seq_list, n, max_context, workspace):
    call("tie_attention_kv4", dtype, q.data_ptr(), q.stride(0), q.shape[0], cache.k_codes.data_ptr(), cache.k_words.data_ptr(), cache.v_codes.data_ptr(),
         cache.v_words.data_ptr(), out.data_ptr(), query_start.data_ptr(), context_lens.data_ptr(), block_tables.data_ptr(), block_tables.shape[1],
         context_lens.numel(), max_queries, q_heads, cache.kv_heads, cache.head_dim, cache.page_size, cache.pages, int(window), float(scale),
         0 if seq_list is None else seq_list.data_ptr(), n, int(max_context), workspace.scratch.data_ptr(), workspace.counters.data_ptr(), _stream())


def attention_kv4_decode(q, cache: Kv4Cache, out, query_start, context_lens, block_tables, q_heads: int, scale: float, seq_list, n_list: int,
                         max_context: int, workspace: Kv4Workspace, window: int = 0) -> None:
    """Attention of sequences that bring one token each over a cache in 4 bits: out[t] for row t = query_start[s] of every sequence s in
    seq_list[:n_list] (int32), over its keys 0..context_lens[s] - 1, the last `window` of them with a window. q [T, >= q_heads * head_dim]
    float32 or bfloat16, out [T, q_heads * head_dim] alike; a sequence without keys gets zeros, other rows are left as they are.
    `max_context`: about the longest of the contexts (how the launch is cut, not what it computes), so that a captured call stays right
    as contexts grow. Softmax statistics and sums are 32-bit; the weights enter the value product with 16 bits (float32 rows: 24)."""
    what = "attention_kv4_decode"
    dtype = _check_attention(what, q, cache, out, query_start, context_lens, block_tables, q_heads, workspace, window, n_list, scale,
                             max_context, 1, seq_list)
    if n_list == 0 or q.shape[0] == 0:
        return
    _rows_kernel(dtype, q, cache, out, query_start, context_lens, block_tables, 1, q_heads, scale, window, seq_list, n_list, min(int(max_context), 2 ** 30), workspace)


def attention_kv4_prompt(q, cache: Kv4Cache, out, query_start, context_lens, block_tables, n_seqs: int, max_queries: int, q_heads: int, scale: float,
                         max_context: int, workspace: Kv4Workspace, window: int = 0) -> None:
    """Causal attention of the first n_seqs sequences of the step, each bringing up to max_queries tokens that are in the cache already: row t of
    sequence s sits at pos = context_lens[s] - (its queries) + (t - query_start[s]) and sees keys 0..pos (with a window: the last `window` of
    them). Types, layouts and `max_context` as in `attention_kv4_decode`."""
    what = "attention_kv4_prompt"
    dtype = _check_attention(what, q, cache, out, query_start, context_lens, block_tables, q_heads, workspace, window, n_seqs, scale,
                             max_context, max_queries)
    max_queries = min(max_queries, q.shape[0])
    if n_seqs == 0 or max_queries == 0:
        return
    _rows_kernel(dtype, q, cache, out, query_start, context_lens, block_tables, max_queries, q_heads, scale, window, None, n_seqs, min(int(max_context), 2 ** 30),
                 workspace)


def step_arrays(n: int, rows: int, columns: int, device="cuda") -> StepArrays:
    """Room for the arrays of a step of n sequences and up to `rows` rows, block tables `columns` pages wide."""
    _need(n >= 0 and rows >= 0 and columns > 0, f"step_arrays: bad sizes ({n} sequences, {rows} rows, {columns} columns)")

    def empty(*shape):
        return torch.empty(*shape, dtype=torch.int32, device=device)
    return StepArrays(empty(n + 1), empty(n), empty(rows), empty(rows), empty(rows), empty(n, columns), empty(1), empty(1))


def _check_tables(what, requests, lens, tables, free_pages, free_count, page_size) -> int:
    _need(requests.dim() == 1 and lens.dim() == 1 and tables.dim() == 2 and free_pages.dim() == 1, f"{what}: requests, lens and free_pages must be 1-D, tables 2-D")
    n = requests.shape[0]
    _int32(what, "requests", requests, n)
    _int32(what, "lens", lens, lens.shape[0])
    _int32(what, "tables", tables, lens.shape[0], tables.shape[1])
    _int32(what, "free_pages", free_pages, free_pages.shape[0])
    _int32(what, "free_count", free_count, 1)
    _need(page_size > 0, f"{what}: page size must be positive")
    return n


def step_tables(requests, counts, lens, tables, free_pages, free_count, page_size: int, arrays: StepArrays, commit: bool = True) -> None:
    """The index arrays of a step from the requests' lengths, all on the GPU (int32 tensors).

    The cache's state: request r holds lens[r] tokens in the pages tables[r, :]; the free pages are a stack, free_pages[:free_count]. Sequence
    i of the step brings counts[i] tokens (zero or more) of request requests[i], no request twice; -1 is padding: its rows get no slot, its context
    is 0. Pages that a request crosses into come off the end of the stack, in the order of the sequences and of their pages, as
    `CacheManager.reserve` hands them out, and are written into `tables`; everything else goes into `arrays` (`step_arrays`), with slot -1,
    position 0 and sequence -1 in the rows behind the last sequence. With `commit` lens and free_count become those after the step; without,
    they stay (a step that is planned again gets the same pages).
    A step that cannot be is refused whole: arrays.status gets the TABLES_* bits that say why (too few free pages; a request longer than
    `tables` or the block tables are wide; more rows than the arrays have; a request outside of lens, a negative count or length, a request
    named twice), every slot is -1, every context and query_start 0, and the state stays as it was."""
    what = "step_tables"
    n = _check_tables(what, requests, lens, tables, free_pages, free_count, page_size)
    rows, columns = arrays.slots.shape[0], arrays.block_tables.shape[-1]
    _int32(what, "counts", counts, n)
    for name, shape in (("query_start", (n + 1,)), ("context_lens", (n,)), ("positions", (rows,)), ("seq_of_row", (rows,)), ("slots", (rows,)),
                        ("block_tables", (n, columns)), ("free_left", (1,)), ("status", (1,))):
        _int32(what, f"arrays.{name}", getattr(arrays, name), *shape)
    _need(0 < columns <= tables.shape[1], f"{what}: block tables of {columns} pages, tables of {tables.shape[1]}")
    _one_device(what, requests, counts, lens, tables, free_pages, free_count, *arrays)
    call("tie_step_tables", requests.data_ptr(), counts.data_ptr(), lens.data_ptr(), tables.data_ptr(), free_pages.data_ptr(), free_count.data_ptr(),
         arrays.query_start.data_ptr(), arrays.context_lens.data_ptr(), arrays.positions.data_ptr(), arrays.seq_of_row.data_ptr(), arrays.slots.data_ptr(),
         arrays.block_tables.data_ptr(), arrays.free_left.data_ptr(), arrays.status.data_ptr(), n, rows, columns, tables.shape[1], lens.shape[0],
         free_pages.shape[0], page_size, 1 if commit else 0, _stream())


def release_tables(requests, lens, tables, free_pages, free_count, page_size: int, status) -> None:
    """The pages of `requests` (int32, no request twice, -1 is skipped) go back onto the end of the stack, the requests in their order and each one's
    pages in theirs, as `CacheManager.release` gives them back; their lengths become 0. Refused whole, with the TABLES_* bits in `status`
    (int32 [1], else 0), where a request or length cannot be or the stack would overflow."""
    what = "release_tables"
    n = _check_tables(what, requests, lens, tables, free_pages, free_count, page_size)
    _int32(what, "status", status, 1)
    _one_device(what, requests, lens, tables, free_pages, free_count, status)
    call("tie_release_tables", requests.data_ptr(), lens.data_ptr(), tables.data_ptr(), free_pages.data_ptr(), free_count.data_ptr(), status.data_ptr(), n,
         lens.shape[0], tables.shape[1], free_pages.shape[0], page_size, _stream())
