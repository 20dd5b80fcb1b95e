"""Keys of the prefill and mixed step graphs over a 4-bit pool, whose attention copies the history: one more part,
the columns of history, and no graph for a copy past the limit (CPU, no device)."""

from types import SimpleNamespace

import pytest

from mini_infra_b200.worker import mixed_graphs as mg
from mini_infra_b200.worker.paged_runner import PagedRunner


def graph_set(block_bytes, wc=2048, bs=16):
    g = object.__new__(mg.MixedGraphSet)
    g.wd = g.wc = wc
    g.pad_token_id, g.max_graphs, g.capture_after = 0, 64, 1
    g.pool = SimpleNamespace(block_size=bs)
    g.history_block_bytes = block_bytes
    g._graphs, g._seen = {}, {}
    g._capture = lambda key: key
    return g


def test_keys_take_the_history_not_the_table():
    g = graph_set(64 << 10)
    assert g.key_for(0, 1, 128, 0, 2048, 0) == (0, 1, 128, 0)
    assert g.key_for(3, 2, 128, 9, 2048, 1) == (4, 2, 128, 16)
    assert g.key_for(3, 2, 128, 9, 2048, 64) == (4, 2, 128, 64)
    assert g.key_for(0, 1, 128, 0, 2048, 65) == (0, 1, 128, 256)
    assert g.key_for(0, 1, 128, 0, 2048, 2000) == (0, 1, 128, 2048)  # 128 MiB
    assert g.key_for(0, 1, 128, 0, 100) == (0, 1, 128, 256)  # no history given: the table's
    assert g.key_for(0, 1, 128, 0, 2049, 0) is None
    narrow = graph_set(64 << 10, wc=32)
    assert narrow.key_for(0, 1, 32, 0, 32, 20) == (0, 1, 32, 32)
    dense = graph_set(0)
    assert dense.key_for(0, 1, 128, 0, 2048, 100) == (0, 1, 128)


@pytest.mark.parametrize("rows", [1, 2, 5, 16, 32])
def test_no_graph_keeps_a_copy_past_the_limit(rows):
    block = 64 << 10  # 16 tokens, 8 heads of 128, K and V in 16 bits
    g = graph_set(block)
    for history in (0, 1, 16, 17, 64, 200, 300, 1024, 2048):
        key = g.key_for(0, rows, 128, 0, 2048, history)
        columns = next(c for c in (*mg.HISTORY_BUCKETS[:-1], 2048) if c >= history)
        held = g.key_for(0, rows, 128, 0, 2048, 0)[1] * columns * block
        assert (key is None) == (held > mg.MAX_HISTORY_BYTES)
        if key is not None:
            assert key[3] == columns >= history
    assert g.key_for(0, rows, 128, 0, 2048, 0) is not None


def test_a_wider_graph_serves_where_none_more_is_captured():
    g = graph_set(64 << 10)
    g.max_graphs = 2
    small, wide, other = (g.key_for(0, 1, 128, 0, 2048, h) for h in (10, 200, 20))
    assert g.consider(wide) and g.consider(small) and g.serving(small) == small
    assert g.consider(other) and g.serving(other) == wide and not g.has(other)
    beyond, longer = g.key_for(0, 1, 128, 0, 2048, 300), g.key_for(0, 1, 256, 0, 2048, 10)
    assert not g.consider(beyond) and g.serving(beyond) is None and not g.consider(longer)


def test_the_runner_counts_history_in_blocks():
    runner = object.__new__(PagedRunner)
    runner.mixed_graphs = g = graph_set(64 << 10)
    kp = SimpleNamespace(data_ptr=lambda: 1)
    g.kv_pools = [(kp, kp)]
    pool = SimpleNamespace(kv_pools=[(kp, kp)], block_size=16)
    tables = [list(range(1, 81)), list(range(81, 100))]
    chunks = [[1] * 40, [2] * 7]
    assert runner._mixed_key([], chunks, tables, pool, [0, 0]) == (0, 2, 64, 0)
    assert runner._mixed_key([], chunks, tables, pool, [0, 256]) == (0, 2, 64, 16)
    assert runner._mixed_key([], chunks, tables, pool, [257, 0]) == (0, 2, 64, 64)
    assert runner._mixed_key([], chunks, tables, pool, None) == (0, 2, 64, 256)
