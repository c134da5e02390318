"""The cache in 4 bits and its step tables, restated in numpy: the quantisation in the 32-bit operations that define it, attention in 64 bits,
the tables through the host's cache manager."""
import numpy as np

from tiny_inference_engine_b200.cache import CacheManager


def padded(head_dim):
    return -(-head_dim // 64) * 64


def quantise(k, v):
    """float32 [..., head_dim] -> ((codes, words) of keys, of values)."""
    with np.errstate(invalid="ignore"):
        bad = ~((np.abs(k) < 2.0 ** 120).all(-1) & (np.abs(v) < 2.0 ** 120).all(-1))
    out = []
    for x, word in ((k, 0x7fc0), (v, 0)):
        x = np.where(bad[..., None], np.float32(0), x.astype(np.float32))
        x = np.concatenate([x, np.zeros((*x.shape[:-1], padded(x.shape[-1]) - x.shape[-1]), np.float32)], -1)
        g = x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
        lo, hi = np.minimum(g.min(-1), np.float32(0)), np.maximum(g.max(-1), np.float32(0))
        least = np.maximum((hi - lo) / np.float32(15), np.float32(2.0 ** -100))
        bits = (least.view(np.uint32) + np.uint32(0x1fffff)) & np.uint32(0xffe00000)
        s = bits.view(np.float32)
        z = np.rint(-lo / s)
        c = np.clip(np.rint(g / s[..., None]) + z[..., None], 0, 15).astype(np.uint8).reshape(x.shape)
        c = np.where(bad[..., None], np.uint8(0), c)
        w = np.where(bad[..., None], np.uint32(word), (bits >> np.uint32(16)) | z.astype(np.uint32)).astype(np.uint16)
        out.append((c[..., 0::2] | (c[..., 1::2] << 4), w))
    return out


def values(codes, words, head_dim):
    """What codes and words stand for, float64 [..., head_dim]."""
    w = words.astype(np.uint32)
    s = ((w & np.uint32(0xffe0)) << np.uint32(16)).view(np.float32).astype(np.float64)
    c = np.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], 2 * codes.shape[-1]).astype(np.float64)
    with np.errstate(invalid="ignore"):
        x = s[..., None] * (c.reshape(*c.shape[:-1], c.shape[-1] // 32, 32) - (w & 15).astype(np.float64)[..., None])
    return x.reshape(c.shape)[..., :head_dim]


def attention(q, k, v, pos, scale, window=0):
    """One head: q [n, d], k and v [keys, d] in 64 bits, pos [n]; rows without keys are zero."""
    key = np.arange(len(k))
    seen = key[None, :] <= pos[:, None]
    if window:
        seen &= key[None, :] > pos[:, None] - window
    out = np.zeros((len(q), v.shape[1]))
    for i in range(len(q)):
        at = np.flatnonzero(seen[i])
        if not len(at):
            continue
        s = scale * (k[at] @ q[i])
        p = np.exp(s - s.max())
        out[i] = (p / p.sum()) @ v[at]
    return out


class HostTables:
    """The state that `step_tables` keeps on the GPU, kept by the host's cache manager (one group, full)."""

    def __init__(self, pages, page_size):
        need = type("Need", (), dict(kind="full", kv_heads=1, head_dim=1, window=0, value_dim=0, keep_first=0))()
        self.manager = CacheManager([need], page_size, num_pages=pages)
        self.page_size = page_size
        self.requests, self.lens = {}, {}

    def step(self, requests, counts, rows, columns):
        """The arrays of a step that can be, as numpy."""
        n = len(requests)
        query_start = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        context = np.zeros(n, np.int32)
        positions, seq_of_row, slots = np.zeros(rows, np.int32), np.full(rows, -1, np.int32), np.full(rows, -1, np.int32)
        tables = np.zeros((n, columns), np.int32)
        for i, (r, c) in enumerate(zip(requests, counts)):
            a, b = query_start[i], query_start[i + 1]
            seq_of_row[a:b] = i
            if r < 0:
                continue
            req = self.requests.setdefault(r, self.manager.new_request())
            held = self.lens.get(r, 0)
            assert self.manager.reserve(req, held + c)
            positions[a:b] = np.arange(held, held + c)
            slots[a:b] = self.manager.slots(req, 0, held, held + c)
            context[i] = self.lens[r] = held + c
            t = req.tables[0]
            tables[i, :len(t)] = t.view()
        return dict(query_start=query_start, context_lens=context, positions=positions, seq_of_row=seq_of_row, slots=slots, block_tables=tables,
                    free_left=np.array([self.manager.num_free()], np.int32), status=np.zeros(1, np.int32))

    def release(self, requests):
        for r in requests:
            if r >= 0 and r in self.requests:
                self.manager.release(self.requests.pop(r))
                self.lens.pop(r, None)
