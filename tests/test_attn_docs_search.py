"""The search for documents of masked attention over long sequences, restated on the CPU
(docs_search.py) and compared with what rows see by definition."""
import numpy as np
import pytest

from docs_search import Warp, documents


def _tiles(n, rows, some):
    starts = np.arange(0, n, rows)
    return [int(i) for i in starts[np.unique(np.linspace(0, len(starts) - 1, some).round().astype(int))]]


def _check(warp, n, tile_rows, some=8, parts=1):
    for i0 in _tiles(n, tile_rows, some):
        visits = [v for part in range(parts) for v in warp.tile(i0, part, parts)]
        for chunk, docs in visits:
            assert docs == tuple(warp.true[chunk]), (i0, chunk)
        assert (warp.seen(i0, visits) == warp.wanted(i0)).all(), i0


@pytest.mark.parametrize("keys", [300, 16385, 20000, 24577, 40000])
@pytest.mark.parametrize("chunk", [64, 96])
@pytest.mark.parametrize("kind", ["runs", "far", "gaps", "shuffled"])
@pytest.mark.parametrize("window", [(-1, -1), (-1, 0)])
def test_documents_of_long_rows(keys, chunk, kind, window):
    """More chunks than the cache of ranges has slots: each visited chunk keeps its own range while
    the search for the next one runs on."""
    doc = documents(keys, kind)
    _check(Warp(doc, doc, chunk, 128, window), keys, 128)


@pytest.mark.parametrize("rows,keys,parts", [(200, 140000, 8), (130, 70000, 4)])
def test_documents_of_few_rows(rows, keys, parts):
    """The keys of a tile divided among blocks, each of which passes more chunks than there are slots."""
    doc = documents(keys, "runs")
    doc_q = doc[np.linspace(0, keys - 1, rows).astype(int)]
    _check(Warp(doc_q, doc, 64, 64), rows, 64, parts=parts)


JUMPS = [  # (window, prefix, the nearest chunk first): positions that are not neighbouring chunks
    ((-1, -1), 0, True), ((-1, 0), 0, True), ((1024, 0), 100, False), ((1024, 0), 1000, False), ((1024, 0), 1000, True),
    ((300, 300), 9000, True), ((300, 5), 16380, False),
]


@pytest.mark.parametrize("keys", [500, 16385, 17000, 20000, 33500])
@pytest.mark.parametrize("chunk", [64, 96])
@pytest.mark.parametrize("window,prefix,near_first", JUMPS)
@pytest.mark.parametrize("kind", ["runs", "shuffled"])
def test_search_ends_where_positions_jump(keys, chunk, window, prefix, near_first, kind):
    """Two of a step's 32 positions may want the same slot for chunks 256 apart."""
    doc = documents(keys, kind)
    warp = Warp(doc, doc, chunk, 128, window, prefix, near_first)
    _check(warp, keys, 128)
    assert warp.filled <= 7  # 32 positions in up to two runs, each of which may begin inside a block
