"""A key/value cache in 4 bits whose step tables are built on the GPU: Python faces of csrc/kv4_cache.cu, csrc/attention_kv4.cu,
csrc/attention_prompt_umma.cu and csrc/step_tables.cu (checks of the arguments, then one or two launches on the current stream).

A token's key (and value) of one kv head is `head_dim` numbers, padded with zeros to whole 64s, in groups of 32. Of a group, with
lo = min(0, its least) and hi = max(0, its largest):

    s = (hi - lo) / 15 in 32 bits, at least 2^-100, rounded up to three significant bits
    z = round(-lo / s),   code = clamp(round(x / s) + z, 0, 15)     (ties to even),   what it stands for: s (code - z)

so that every value is a bfloat16 number within s of what was appended, and costs 4.5 bits. Codes lie in padded / 2 bytes, dimension d in
byte d // 2, the even one in the low bits; a group's 16-bit word holds s as bfloat16 (its low five bits are zero) and z in its low four. A token
and head whose key or value holds a number that is not finite, or one of magnitude 2^120 or more, gets the key words 0x7fc0, zero
value words and zero codes: rows that see that key are NaN, no other is. Attention sees the values that `kv4_read` gives, over the whole range of
steps (from 2^26 on, which no model's keys come near, with a product more a value).
"""
from __future__ import annotations

import os
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


class Kv4Workspace:
    """Where the splits of a row's keys leave their sums: `scratch` float32 (contiguous, 16-byte aligned), `counters` int32 zeros
    (`kv4_workspace_sizes`), looked over once, here. Calls that run one after the other may share a workspace (its counters are zero between
    them); calls that may run at the same time, in two streams or two captured graphs, need one each."""
    __slots__ = ("scratch", "counters", "floats", "ctas", "pointers", "device")

    def __init__(self, scratch: torch.Tensor, counters: torch.Tensor):
        if scratch.dtype is not torch.float32 or counters.dtype is not torch.int32 or not (scratch.is_contiguous() and counters.is_contiguous()) or \
                scratch.data_ptr() & 15 or scratch.get_device() != counters.get_device():
            raise InvalidArgument("Kv4Workspace: scratch must be contiguous float32, 16-byte aligned, counters contiguous int32, both on one device")
        self.scratch, self.counters = scratch, counters
        self.floats, self.ctas, self.device = scratch.numel(), counters.numel(), scratch.get_device()
        self.pointers = scratch.data_ptr(), counters.data_ptr()


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


# The checks run on every call, ahead of kernels of a few microseconds: conditions are tested in plain `if`s, so that a message is only put
# together when it is needed, and every property of a tensor is asked for once.

def _need(cond, msg: str) -> None:
    if not cond:
        raise InvalidArgument(msg)


def _fail(msg: str):
    raise InvalidArgument(msg)


# When the tcgen05 kernel takes the portions of a prompt, in place of the one whose warps take 16 rows each: from UMMA_MIN_ROWS rows (queries x heads
# of a group) a portion, and UMMA_GROUPS of 16 rows in all, or with long contexts UMMA_FEW_GROUPS (groups x keys UMMA_GROUPS x 1,024). It starts
# slower (9 to 15 us a call against 5 to 10) and its tiles of 128 rows are too few for the GPU until then. bfloat16, 32 heads over 8 of 128, us with
# it and without: 64 portions of 16 rows at 512 keys 62 and 27, 32 of 48 rows at 64 16 and 23, 16 of 64 rows 9 and 16; one of 64 queries at 300 keys (128
# groups) 15 and 11, 128 at 1,024 (256 groups) 27 and 22, at 2,048 34 and 47, 192 at 1,024 (384 groups) 26 and 36, 512 at 512 17 and 38; 4
# of 512 at 2,048 91 and 406. float32: 64 at 300 20 and 11, 192 at 1,024 33 and 45, 4 of 512 at 2,048 195 and 656.
UMMA_MIN_ROWS, UMMA_GROUPS, UMMA_FEW_GROUPS = 48, 384, 128
_NO_UMMA_ATTENTION = os.environ.get("TIE_NO_UMMA_ATTENTION") == "1"
_FLOATS = {torch.float32: 0, torch.bfloat16: 1}
_I32 = torch.int32


def _stream(what: str, *ts) -> int:
    """The current stream, once every tensor is known to be on the current device."""
    here = _CURRENT_DEVICE() if ts[0].is_cuda else -1
    for t in ts:
        if t.get_device() != here or here < 0:
            _fail("kernel arguments must be CUDA tensors: the engine has no CPU path" if not t.is_cuda else
                  f"{what}: all tensors must be on the current device, {here}, got one on {t.device}")
    return _RAW_STREAM(here)


_CURRENT_DEVICE, _RAW_STREAM = getattr(torch._C, "_cuda_getDevice", None), getattr(torch._C, "_cuda_getCurrentRawStream", None)


def kv4_cache(pages: int, kv_heads: int, page_size: int, head_dim: int, device="cuda") -> Kv4Cache:
    """An empty cache for one layer (of any number of requests)."""
    _need(pages > 0 and kv_heads > 0 and page_size > 0 and 0 < head_dim <= 256 and pages * kv_heads * page_size < 2 ** 31,
          f"kv4_cache: bad sizes (pages {pages}, kv heads {kv_heads}, page size {page_size}, head size {head_dim}, at most 256)")
    padded = -(-head_dim // 64) * 64

    def plane(width, dtype):
        return torch.zeros(pages, kv_heads, page_size, width, dtype=dtype, device=device)
    return Kv4Cache(plane(padded // 2, torch.uint8), plane(padded // 32, torch.int16), plane(padded // 2, torch.uint8), plane(padded // 32, torch.int16), head_dim)


def _check_cache(what: str, c: Kv4Cache) -> tuple:
    """The planes' addresses and (kv heads, head size, page size, pages)."""
    kc, kw, vc, vw, dim = c
    if not 0 < dim <= 256:
        _fail(f"{what}: head size {dim} is not in 1..256")
    words = (dim + 63) // 64 * 2
    shape = kc.shape
    if len(shape) != 4:
        _fail(f"{what}: codes must be [pages, kv_heads, page_size, bytes]")
    pages, heads, size, width = shape
    n = pages * heads * size * words
    if width != 16 * words or not (kc.dtype is vc.dtype is torch.uint8 and kw.dtype is vw.dtype is torch.int16) or kw.numel() != n or vw.numel() != n or \
            vc.numel() != 16 * n or not (kc.is_contiguous() and kw.is_contiguous() and vc.is_contiguous() and vw.is_contiguous()):
        _fail(f"{what}: planes must be contiguous, codes uint8 [pages, kv_heads, page_size, {16 * words}] and words int16 [..., {words}]")
    if n == 0 or pages * heads * size >= 2 ** 31:
        _fail(f"{what}: planes must have one row at least and less than 2^31 (pages x kv heads x page size)")
    planes = kc.data_ptr(), kw.data_ptr(), vc.data_ptr(), vw.data_ptr()
    if (planes[0] | planes[1] | planes[2] | planes[3]) & 15:
        _fail(f"{what}: planes must be 16-byte aligned")
    return planes, (heads, dim, size, pages)


def _check_rows(what: str, c: Kv4Cache, k, v, slots, written=False) -> tuple:
    planes, sizes = _check_cache(what, c)
    dtype = _FLOATS.get(k.dtype)
    if dtype is None or v.dtype is not k.dtype:
        _fail(f"{what}: rows must be float32 or bfloat16, all alike")
    shape, width = k.shape, sizes[0] * sizes[1]
    if len(shape) != 2 or shape[1] != width or v.shape != shape:
        _fail(f"{what}: k and v must be [T, {width}]")
    (k_stride, k_step), (v_stride, v_step) = k.stride(), v.stride()
    if (k_step != 1 or v_step != 1) and width > 1:
        _fail(f"{what}: k and v must be [T, {width}] with contiguous rows")
    if written and shape[0] > 1 and (k_stride < width or v_stride < width):
        _fail(f"{what}: rows of k and v must not overlap")
    if slots.dtype is not _I32 or slots.numel() != shape[0] or not slots.is_contiguous():
        _fail(f"{what}: slots must be contiguous int32 [{shape[0]}]")
    return dtype, planes, sizes, shape[0], k_stride, v_stride, _stream(what, k, v, slots, c[0], c[1], c[2], c[3])


def kv4_append(k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, cache: Kv4Cache) -> None:
    """k, v [T, kv_heads * head_dim] (float32 or bfloat16, rows may be strided) into the cache at slots[t]; slot < 0 writes nothing. The slots of a
    call must differ: of a slot that is named twice it is not said which row it keeps, or which part of either. A slot outside of the cache
    writes nothing either and is reported by `gemm_select.check_status`."""
    dtype, planes, sizes, T, k_stride, v_stride, stream = _check_rows("kv4_append", cache, k, v, slots)
    call("tie_kv4_append", dtype, k.data_ptr(), v.data_ptr(), k_stride, v_stride, slots.data_ptr(), *planes, T, *sizes, stream)


def kv4_read(cache: Kv4Cache, slots: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> None:
    """The values that the cache holds at slots[t] into k, v [T, kv_heads * head_dim] (float32 or bfloat16, exact in both); rows whose slot is below
    zero are left as they are. Rows of one tensor must not overlap."""
    dtype, planes, sizes, T, k_stride, v_stride, stream = _check_rows("kv4_read", cache, k, v, slots, True)
    call("tie_kv4_read", dtype, *planes, slots.data_ptr(), k.data_ptr(), v.data_ptr(), k_stride, v_stride, T, *sizes, stream)


def kv4_workspace_sizes(head_dim: int) -> tuple[int, int]:
    """(float32 numbers, int32 zeros) of a workspace for heads of this size: for callers that keep buffers of their own (both contiguous,
    16-byte aligned)."""
    ctas = _workspace_ctas()
    return ctas * 16 * (-(-head_dim // 64) * 64 + 2), ctas


def kv4_workspace(q_heads: int, kv_heads: int, head_dim: int, device="cuda") -> Kv4Workspace:
    """The workspace of `attention_kv4_decode` and `attention_kv4_prompt` for heads of these sizes, whatever the batch."""
    _need(q_heads > 0 and kv_heads > 0 and q_heads % kv_heads == 0 and 0 < head_dim <= 256, "kv4_workspace: bad sizes")
    floats, counters = kv4_workspace_sizes(head_dim)
    return Kv4Workspace(torch.empty(floats, dtype=torch.float32, device=device), torch.zeros(counters, dtype=torch.int32, device=device))


def _workspace_ctas() -> int:
    global _CTAS
    if _CTAS is None:
        _CTAS = library().tie_attention_kv4_ctas()
    return _CTAS


_CTAS = None        # CTAs that may leave partial sums: what the kernels were compiled for


def _check_attention(what, q, cache, out, query_start, context_lens, block_tables, q_heads, workspace, window, n: int, scale, max_context,
                     max_queries: int, seq_list=None) -> tuple:
    """(dtype, the planes' addresses, their sizes, rows, row stride of q, sequences, columns of the block tables, stream)"""
    planes, sizes = _check_cache(what, cache)
    dtype = _FLOATS.get(q.dtype)
    if dtype is None or out.dtype is not q.dtype:
        _fail(f"{what}: rows must be float32 or bfloat16, all alike")
    if q_heads <= 0 or q_heads % sizes[0]:
        _fail(f"{what}: {q_heads} heads are not a multiple of {sizes[0]} kv heads")
    width, shape, out_shape, table_shape = q_heads * sizes[1], q.shape, out.shape, block_tables.shape
    if len(shape) != 2 or shape[1] < width:
        _fail(f"{what}: q must be [T, {width}] or wider")
    q_stride, step = q.stride()
    if step != 1 and shape[1] > 1:
        _fail(f"{what}: q must have contiguous rows")
    if len(out_shape) != 2 or out_shape[0] != shape[0] or out_shape[1] != width or not out.is_contiguous():
        _fail(f"{what}: out must be contiguous [T, {width}]")
    S = context_lens.numel()
    if not (query_start.dtype is context_lens.dtype is block_tables.dtype is _I32) or query_start.numel() != S + 1 or len(table_shape) != 2 or \
            table_shape[0] != S or not (query_start.is_contiguous() and context_lens.is_contiguous() and block_tables.is_contiguous()):
        _fail(f"{what}: query_start [{S + 1}], context_lens [{S}] and block_tables [{S}, pages] must be contiguous int32")
    if not 0 <= n <= 65535 or (seq_list is None and n > S):
        _fail(f"{what}: {n} of {S} sequences (at most 65,535 a call)")
    if not 0 <= window < 2 ** 30:
        _fail(f"{what}: bad window {window}")
    ctas = _workspace_ctas()
    if workspace.floats < ctas * 16 * ((sizes[1] + 63) // 64 * 64 + 2) or workspace.ctas < ctas:
        _fail(f"{what}: the workspace is too small (kv4_workspace makes one)")
    if not (scale > 0 and max_context >= 0 and 0 <= max_queries < 2 ** 30):
        _fail(f"{what}: the scale must be positive, max_context and max_queries not negative")
    if seq_list is None:
        stream = _stream(what, q, out, query_start, context_lens, block_tables, cache[0], cache[1], cache[2], cache[3])
    else:
        if seq_list.dtype is not _I32 or seq_list.dim() != 1 or not seq_list.is_contiguous() or seq_list.numel() < n:
            _fail(f"{what}: seq_list must be int32 [n_list]")
        stream = _stream(what, q, out, query_start, context_lens, block_tables, cache[0], cache[1], cache[2], cache[3], seq_list)
    if workspace.device != q.get_device():
        _fail(f"{what}: the workspace must be on the current device")
    return dtype, planes, sizes, shape[0], q_stride, S, table_shape[1], stream


def _rows_kernel(checked, q, out, query_start, context_lens, block_tables, max_queries, q_heads, scale, window, seq_list, n, max_context, workspace):
    dtype, planes, sizes, T, q_stride, S, columns, stream = checked
    call("tie_attention_kv4", dtype, q.data_ptr(), q_stride, T, *planes, out.data_ptr(), query_start.data_ptr(), context_lens.data_ptr(),
         block_tables.data_ptr(), columns, S, max_queries, q_heads, *sizes, window, scale, seq_list, n, min(max_context, 2 ** 30),
         *workspace.pointers, stream)


def attention_kv4_decode(q, cache: Kv4Cache, out, query_start, context_lens, block_tables, q_heads: int, scale: float, seq_list, n_list: int,
                         max_context: int, workspace: Kv4Workspace, window: int = 0) -> None:
    """Attention of sequences that bring one token each over a cache in 4 bits: out[t] for row t = query_start[s] of every sequence s in
    seq_list[:n_list] (int32), over its keys 0..context_lens[s] - 1, the last `window` of them with a window. q [T, >= q_heads * head_dim]
    float32 or bfloat16, out [T, q_heads * head_dim] alike; a sequence without keys gets zeros, other rows are left as they are.
    `max_context`: about the longest of the contexts (how the launch is cut, not what it computes), so that a captured call stays right
    as contexts grow. Softmax statistics and sums are 32-bit; the weights enter the value product with 16 bits (float32 rows: 24)."""
    checked = _check_attention("attention_kv4_decode", q, cache, out, query_start, context_lens, block_tables, q_heads, workspace, window, n_list, scale,
                               max_context, 1, seq_list)
    if n_list and checked[3]:
        _rows_kernel(checked, q, out, query_start, context_lens, block_tables, 1, q_heads, scale, window, seq_list.data_ptr(), n_list, max_context, workspace)


def _on_tcgen05(dtype, sizes, T, group, n_seqs, max_queries, keys):
    rows, head_dim = max_queries * group, sizes[1]
    if _NO_UMMA_ATTENTION or rows < UMMA_MIN_ROWS or head_dim > (256 if dtype else 128) or head_dim % 8 or n_seqs > 16383 or rows > 65535 * 128:
        return False
    groups = sizes[0] * min(n_seqs * ((rows + 15) // 16), T * group // 16 + n_seqs)
    return groups >= UMMA_GROUPS or (groups >= UMMA_FEW_GROUPS and groups * keys >= UMMA_GROUPS * 1024)


def attention_kv4_prompt(q, cache: Kv4Cache, out, query_start, context_lens, block_tables, n_seqs: int, max_queries: int, q_heads: int, scale: float,
                         max_context: int, workspace: Kv4Workspace, window: int = 0) -> None:
    """Causal attention of the first n_seqs sequences of the step, each bringing up to max_queries tokens that are in the cache already: row t of
    sequence s sits at pos = context_lens[s] - (its queries) + (t - query_start[s]) and sees keys 0..pos (with a window: the last `window` of
    them). A sequence that brings more than max_queries tokens has its first ones only, the other rows are left as they are. Types, layouts and
    `max_context` as in `attention_kv4_decode`; long portions (`UMMA_MIN_ROWS` and what stands there; 16-byte aligned rows, heads of a multiple of 8
    up to 256, float32 128) run on tcgen05, where the weights of bfloat16 rows enter the value product as one bfloat16 number."""
    checked = _check_attention("attention_kv4_prompt", q, cache, out, query_start, context_lens, block_tables, q_heads, workspace, window, n_seqs, scale,
                               max_context, max_queries)
    max_queries = min(max_queries, checked[3])
    if not n_seqs or not max_queries:
        return
    dtype, planes, sizes, T, q_stride, _, columns, stream = checked
    if _on_tcgen05(dtype, sizes, T, q_heads // sizes[0], n_seqs, max_queries, min(max_context, window + max_queries) if window else max_context) and \
            q_stride % (8 if dtype else 4) == 0 and not (q.data_ptr() | out.data_ptr()) & 15:
        call("tie_attention_prompt_kv4", dtype, q.data_ptr(), q_stride, T, *planes, out.data_ptr(), query_start.data_ptr(), context_lens.data_ptr(),
             block_tables.data_ptr(), columns, n_seqs, max_queries, q_heads, *sizes, window, scale, min(max_context, 2 ** 30), stream)
    else:
        _rows_kernel(checked, q, out, query_start, context_lens, block_tables, max_queries, q_heads, scale, window, 0, n_seqs, max_context, workspace)


def step_arrays(n: int, rows: int, columns: int, device="cuda") -> StepArrays:
    """Room for the arrays of a step of n sequences and up to `rows` rows, block tables `columns` pages wide."""
    _need(n >= 0 and rows >= 0 and columns > 0, f"step_arrays: bad sizes ({n} sequences, {rows} rows, {columns} columns)")

    def empty(*shape):
        return torch.empty(*shape, dtype=torch.int32, device=device)
    return StepArrays(empty(n + 1), empty(n), empty(rows), empty(rows), empty(rows), empty(n, columns), empty(1), empty(1))


def _check_tables(what, requests, lens, tables, free_pages, free_count, page_size) -> tuple:
    """(sequences, requests of the state, columns of its tables, pages)"""
    shape, n, held, pages = tables.shape, requests.numel(), lens.numel(), free_pages.numel()
    if not (requests.dtype is lens.dtype is free_pages.dtype is free_count.dtype is tables.dtype is _I32) or free_count.numel() != 1 or len(shape) != 2 or \
            shape[0] != held or not (requests.is_contiguous() and lens.is_contiguous() and free_pages.is_contiguous() and tables.is_contiguous()):
        _fail(f"{what}: requests, lens [{held}], tables [{held}, pages], free_pages and free_count [1] must be contiguous int32")
    if page_size <= 0:
        _fail(f"{what}: page size must be positive")
    return n, held, shape[1], pages


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
    named twice), every slot is -1, every context and query_start 0, and the state stays as it was. At most 8,192 sequences of 131,072 requests."""
    what = "step_tables"
    n, held, width, pages = _check_tables(what, requests, lens, tables, free_pages, free_count, page_size)
    query_start, context_lens, positions, seq_of_row, slots, block_tables, free_left, status = arrays
    rows, shape = slots.numel(), block_tables.shape
    if not (counts.dtype is query_start.dtype is context_lens.dtype is positions.dtype is seq_of_row.dtype is slots.dtype is block_tables.dtype is
            free_left.dtype is status.dtype is _I32) or counts.numel() != n or query_start.numel() != n + 1 or context_lens.numel() != n or \
            positions.numel() != rows or seq_of_row.numel() != rows or free_left.numel() != 1 or status.numel() != 1 or not (
            counts.is_contiguous() and query_start.is_contiguous() and context_lens.is_contiguous() and positions.is_contiguous() and
            seq_of_row.is_contiguous() and slots.is_contiguous()):
        _fail(f"{what}: counts [{n}] and arrays (step_arrays makes them for {n} sequences) must be contiguous int32")
    if len(shape) != 2 or shape[0] != n or not block_tables.is_contiguous() or not 0 < shape[1] <= width:
        _fail(f"{what}: arrays.block_tables must be contiguous [{n}, up to {width}]")
    stream = _stream(what, requests, counts, lens, tables, free_pages, free_count, query_start, context_lens, positions, seq_of_row, slots, block_tables,
                     free_left, status)
    call("tie_step_tables", requests.data_ptr(), counts.data_ptr(), lens.data_ptr(), tables.data_ptr(), free_pages.data_ptr(), free_count.data_ptr(),
         query_start.data_ptr(), context_lens.data_ptr(), positions.data_ptr(), seq_of_row.data_ptr(), slots.data_ptr(), block_tables.data_ptr(),
         free_left.data_ptr(), status.data_ptr(), n, rows, shape[1], width, held, pages, page_size, 1 if commit else 0, stream)


def release_tables(requests, lens, tables, free_pages, free_count, page_size: int, status) -> None:
    """The pages of `requests` (int32, no request twice, -1 is skipped) go back onto the end of the stack, the requests in their order and each one's
    pages in theirs, as `CacheManager.release` gives them back; their lengths become 0. Refused whole, with the TABLES_* bits in `status`
    (int32 [1], else 0), where a request or length cannot be or the stack would overflow. At most 8,192 of 131,072 requests."""
    what = "release_tables"
    n, held, width, pages = _check_tables(what, requests, lens, tables, free_pages, free_count, page_size)
    if status.dtype is not _I32 or status.numel() != 1:
        _fail(f"{what}: status must be int32 [1]")
    stream = _stream(what, requests, lens, tables, free_pages, free_count, status)
    call("tie_release_tables", requests.data_ptr(), lens.data_ptr(), tables.data_ptr(), free_pages.data_ptr(), free_count.data_ptr(), status.data_ptr(), n,
         held, width, pages, page_size, stream)
