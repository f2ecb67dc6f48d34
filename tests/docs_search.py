"""The search for documents of masked attention's loading warp (csrc/attn_tile.cuh) restated on the
CPU, lane by lane where lanes differ: which chunks of keys a tile visits, in which order, with
which documents, and what its rows then see of them."""
import numpy as np

LANES = np.arange(32)
RANGES = 256  # slots of chunks' ranges, a tag for eight each
NONE = 2**31 - 1


class Warp:
    """A loading warp: its cache of ranges outlives the items of one sequence."""

    def __init__(self, doc_q, doc_k, chunk, tile_rows, window=(-1, -1), prefix=0, near_first=False):
        self.doc_q, self.doc_k, self.kc, self.tile_rows = doc_q, doc_k, chunk, tile_rows
        self.window, self.prefix, self.near_first = window, min(prefix, len(doc_k)), near_first
        n = -(-len(doc_k) // chunk) + 64  # (blocks of eight and steps of 32 end behind the keys)
        keys = np.full(n * chunk, -1)
        keys[: len(doc_k)] = doc_k
        keys = keys.reshape(n, chunk)
        least = np.where(keys < 0, NONE, keys).min(1)
        most = keys.max(1).clip(min=-1)
        self.true = np.stack([least, np.where((keys < 0).any(1), -1 - most.clip(min=0), most)], 1)
        self.tag = np.full(RANGES // 8, -1)
        self.range = np.zeros((RANGES, 2), dtype=np.int64)
        self.filled = 0  # most blocks of eight fetched for a step of 32 positions

    def span(self, place):
        """The window of the row at `place`."""
        m = len(self.doc_k)
        lo = 0 if self.window[0] < 0 else max(place - self.window[0], 0)
        hi = max(m if self.window[1] < 0 else min(place + self.window[1] + 1, m), 0)
        return min(lo, hi), hi

    def fetch(self, block):
        at = np.arange(8 * block, 8 * block + 8)
        self.range[at % RANGES] = self.true[at]
        self.tag[block % (RANGES // 8)] = block

    def tile(self, i0, part=0, parts=1):
        """[(chunk, flags' range of documents)] of the tile whose first row is i0."""
        kc, n, m = self.kc, len(self.doc_q), len(self.doc_k)
        last, shift = min(i0 + self.tile_rows, n) - 1, m - n
        lo0, hi1 = self.span(i0 + shift)[0], self.span(last + shift)[1]
        n1 = -(-self.prefix // kc)
        c0 = max(n1, lo0 // kc)
        total = n1 + (max(-(-hi1 // kc) - c0, 0) if hi1 > self.span(last + shift)[0] else 0)
        end, t = total * (part + 1) // parts, total * part // parts
        turn = 0
        if parts == 1 and self.near_first and total > 0:
            near = max((i0 + last) // 2 + shift, 0) // kc
            turn = 0 if n1 <= near < c0 else min(near if near < c0 else n1 + near - c0, total - 1)

        def chunk_at(p):
            p = p + turn
            p = np.where(p >= total, p - total, p)
            return np.where(p < n1, p, c0 + p - n1)

        docs = self.doc_q[i0 : last + 1]
        docs = docs[docs >= 0]
        dq0, dq1 = (docs.min(), docs.max()) if len(docs) else (NONE, -1)
        hits, hits_at, docs_of = np.zeros(32, dtype=bool), -32, np.zeros((32, 2), dtype=np.int64)

        def seek(at):
            nonlocal hits, hits_at, docs_of
            if at < hits_at + 32:
                ahead = hits[at - hits_at :]
                if ahead.any():
                    return at + int(ahead.argmax())
                at = hits_at + 32
            while at < end:
                p = at + LANES
                c = chunk_at(np.where(p < end, p, at))
                docs_of = self.step(c, p < end)
                most = np.where(docs_of[:, 1] < 0, -1 - docs_of[:, 1], docs_of[:, 1])
                hits, hits_at = (p < end) & (docs_of[:, 0] <= dq1) & (most >= dq0), at
                if hits.any():
                    return at + int(hits.argmax())
                at += 32
            return max(at, end)

        visits, pend = [], None
        while True:  # a chunk is loaded once it is known whether another follows
            t = seek(t)
            found = None
            if t < end:
                found = int(chunk_at(np.int64(t))), tuple(docs_of[t - hits_at])
            if pend is not None:
                visits.append(pend)
            if found is None:
                return visits
            pend, t = found, t + 1

    def step(self, c, on):
        """The ranges of the lanes' chunks c (where `on`): a lane takes its own while its slot holds it."""
        want, got, blocks = on.copy(), np.zeros((32, 2), dtype=np.int64), 0
        while True:
            there = want & (self.tag[(c >> 3) % (RANGES // 8)] == c >> 3)
            got[there] = self.range[c % RANGES][there]
            want &= ~there
            if not want.any():
                break
            self.fetch(int((c >> 3)[want.argmax()]))
            blocks += 1
            assert blocks <= 32, "the search does not end"
        self.filled = max(self.filled, blocks)
        return got

    def seen(self, i0, visits):
        """What the tile's rows see, [rows, keys]: windows and prefix, and documents by the chunk's flags."""
        n, m, kc = len(self.doc_q), len(self.doc_k), self.kc
        rows = np.arange(i0, min(i0 + self.tile_rows, n))
        doc = self.doc_q[rows]
        got = np.zeros((len(rows), m), dtype=bool)
        for c, (least, most) in visits:
            j = slice(c * kc, min(c * kc + kc, m))
            assert not got[:, j].any(), "a chunk twice"
            if least == most:  # one document
                got[:, j] = (doc == least)[:, None]
            else:
                got[:, j] = (doc[:, None] == self.doc_k[j]) & (doc >= 0)[:, None]
        return got & self.placed(rows)

    def placed(self, rows):
        lo, hi = np.array([self.span(int(i) + len(self.doc_k) - len(self.doc_q)) for i in rows]).T
        j = np.arange(len(self.doc_k))
        return ((j >= lo[:, None]) & (j < hi[:, None])) | (j < self.prefix)

    def wanted(self, i0):
        rows = np.arange(i0, min(i0 + self.tile_rows, len(self.doc_q)))
        doc = self.doc_q[rows]
        return (doc[:, None] == self.doc_k) & (doc >= 0)[:, None] & self.placed(rows)


def documents(n, kind, seed=0):
    """Numbers of n keys: "runs" of uneven lengths, "far" (the same number at both ends), "gaps"
    (runs with keys of none among them) or "shuffled"."""
    r = np.random.default_rng(seed + n)
    doc = np.searchsorted(np.sort(r.integers(0, n, 23)), np.arange(n), side="right")
    if kind == "far":
        doc[-100:] = doc[:50].repeat(2)
    if kind == "gaps":
        doc[r.integers(0, n, 40)[:, None] + np.arange(30) - n] = -1
    if kind == "shuffled":
        r.shuffle(doc)
    return doc
