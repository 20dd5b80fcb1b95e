"""Forked and compacted block tables (KVCacheManager.fork / compact), the 4-bit cache's configuration and its
format's oracle: host-side parts, no GPU."""

import ctypes

import numpy as np
import pytest

from mini_infra_b200 import _native as nat
from mini_infra_b200 import ops
from mini_infra_b200.core import KVCacheManager, PagedCacheConfig
from mini_infra_b200.core.types import kv_cache_config_from_str
from oracle import kv4_oracle as ko


class Pages:
    """A stand-in for the pools: what every (block, offset) holds."""

    def __init__(self, manager):
        self.m, self.data = manager, {}

    def write(self, req, start, values):
        for i, v in enumerate(values):
            p = start + i
            self.data[self.m.block_table(req)[p // self.m.block_size], p % self.m.block_size] = v

    def read(self, req, n):
        bs = self.m.block_size
        return [self.data[self.m.block_table(req)[p // bs], p % bs] for p in range(n)]

    def copy(self, pairs):
        old = dict(self.data)
        for s, d in pairs:
            for o in range(self.m.block_size):
                self.data[d, o] = old.get((s, o))


@pytest.mark.parametrize("tokens", [1, 3, 4, 5, 8])
def test_fork_shares_full_blocks_and_copies_the_partial_one(tokens):
    m = KVCacheManager(4, 16)
    pages = Pages(m)
    assert m.allocate_slots(0, tokens)
    pages.write(0, 0, range(tokens))
    used = m.num_used_blocks
    moves = m.fork(0, 1)
    assert len(moves) == (tokens % 4 > 0) and m.num_used_blocks == used + len(moves)
    pages.copy(moves)
    assert pages.read(1, tokens) == list(range(tokens))
    full = tokens // 4
    assert m.block_table(0)[:full] == m.block_table(1)[:full]
    assert set(m.block_table(0)[full:]).isdisjoint(m.block_table(1)[full:])
    for req, mark in ((0, "a"), (1, "b")):  # both go on
        assert m.allocate_slots(req, 3)
        pages.write(req, tokens, [mark] * 3)
    assert pages.read(0, tokens + 3) == [*range(tokens), *"aaa"]
    assert pages.read(1, tokens + 3) == [*range(tokens), *"bbb"]
    m.free(0)
    assert pages.read(1, tokens) == list(range(tokens)) and m.num_used_blocks == len(m.block_table(1))
    m.free(1)
    assert m.num_used_blocks == 0


def test_fork_of_a_fork_frees_with_its_last_holder():
    m = KVCacheManager(2, 10)
    assert m.allocate_slots(0, 4)
    assert m.fork(0, 1) == [] and m.fork(1, 2) == []
    for left, req in ((2, 0), (2, 2), (0, 1)):
        m.free(req)
        assert m.num_used_blocks == left
    assert m.block_release_count == 2


def test_fork_refusals():
    m = KVCacheManager(4, 3)
    assert m.allocate_slots(0, 7)
    with pytest.raises(KeyError):
        m.fork(5, 6)
    with pytest.raises(ValueError):
        m.fork(0, 0)
    table, used = list(m.block_table(0)), m.num_used_blocks
    assert m.fork(0, 1) is None  # the copy's block is not free: nothing changed
    assert m.block_table(0) == table and m.num_used_blocks == used
    with pytest.raises(KeyError):
        m.block_table(1)


def test_compaction_keeps_every_requests_tokens():
    rng = np.random.default_rng(0)
    m = KVCacheManager(4, 200)
    pages, live, n = Pages(m), {}, 0
    for _ in range(400):
        what = rng.integers(0, 10)
        if what < 4 and len(live) < 20:
            n += 1
            k = int(rng.integers(1, 30))
            if m.allocate_slots(n, k):
                live[n] = [int(x) for x in rng.integers(0, 1000, k)]
                pages.write(n, 0, live[n])
        elif what < 6 and live:
            src = int(rng.choice(list(live)))
            n += 1
            moves = m.fork(src, n)
            if moves is not None:
                pages.copy(moves)
                live[n] = list(live[src])
        elif what < 8 and live:
            req = int(rng.choice(list(live)))
            if m.allocate_slots(req, 1):
                live[req].append(int(rng.integers(0, 1000)))
                pages.write(req, len(live[req]) - 1, live[req][-1:])
        elif what == 8 and live:
            req = int(rng.choice(list(live)))
            m.free(req)
            del live[req]
        else:
            used = m.num_used_blocks
            moves = m.compact()
            assert {d for _, d in moves}.isdisjoint({s for s, _ in moves})
            assert all(d <= used < s for s, d in moves)
            pages.copy(moves)
            held = {b for r in live for b in m.block_table(r)}
            assert held == set(range(1, used + 1)) and m.num_used_blocks == used
            assert m.compact() == []
        for req, want in live.items():
            assert pages.read(req, len(want)) == want
    for req in live:
        m.free(req)
    assert m.num_used_blocks == 0
    assert m.allocate_slots(10**6, 4 * 199)
    assert sorted(m.block_table(10**6)) == list(range(1, 200))


def test_device_tables_resend_after_invalidation():
    import torch

    from mini_infra_b200.worker.block_tables import DeviceBlockTables

    t = DeviceBlockTables(2, 4, torch.device("cpu"))
    _, _, d = t.step_inputs([(0, 7)], [[5, 6]], [1], [3])
    assert d == 2
    t.invalidate()
    host, _, d = t.step_inputs([(0, 7)], [[1, 2]], [1], [3])
    assert d == 2 and host[3:].tolist() == [0, 0, 1, 0, 1, 2]


def test_cache_config():
    assert PagedCacheConfig().kv_bits == 16 and str(PagedCacheConfig()) == "paged-kv-cache(block_size=16)"
    assert str(PagedCacheConfig(kv_bits=4)) == "paged-kv-cache(block_size=16,kv_bits=4)"
    assert kv_cache_config_from_str("paged-kv-cache", kv_bits=4).kv_bits == 4
    with pytest.raises(ValueError):
        PagedCacheConfig(kv_bits=8)


def test_page_bytes():
    lib = nat.load()
    for bs, d in ((16, 128), (1, 32), (3, 96), (32, 256)):
        assert lib.mi_kv4_page_bytes(bs, d) == ops.kv4_page_bytes(bs, d) == ko.page_bytes(bs, d)
    for bs, d in ((0, 128), (16, 0), (16, 48), (16, 288)):
        assert lib.mi_kv4_page_bytes(bs, d) == 0
        with pytest.raises(ValueError):
            ops.kv4_page_bytes(bs, d)


def test_host_rejects_bad_arguments_before_launch():
    """No pointer is touched: every call is refused by a check of sizes or for a null pointer."""
    lib = nat.load()
    s = nat.i64_array([0, 0, 0])
    fine = ctypes.c_void_p(256)  # never read: the checks before it fail

    def scatter(n=4, bs=16, d=128, blocks=8, dtype=nat.MI_BF16, pool=None, src=None):
        return lib.mi_kv4_scatter(src, src, s, s, 4, 1, None, None, None, n, pool, pool, blocks, bs, 8, d, dtype, None)

    assert scatter() == nat.MI_ERR_INVALID and "null pointer" in nat.last_error()
    assert scatter(dtype=7) == nat.MI_ERR_INVALID and "dtype" in nat.last_error()
    assert scatter(d=100) == nat.MI_ERR_INVALID and "multiple of 32" in nat.last_error()
    assert scatter(n=-1) == nat.MI_ERR_INVALID
    assert scatter(pool=ctypes.c_void_p(258)) == nat.MI_ERR_INVALID and "aligned" in nat.last_error()
    assert scatter(blocks=1 << 28) == nat.MI_ERR_UNSUPPORTED
    assert scatter(n=0) == nat.MI_OK

    def chunks(batch=2, length=4, width=3, stride=3):
        return lib.mi_kv4_store_chunks(fine, fine, s, s, batch, length, fine, fine, fine, stride, width, fine, fine, 8, 16,
                                       8, 128, nat.MI_BF16, None)

    assert chunks(stride=2) == nat.MI_ERR_INVALID and "stride" in nat.last_error()
    assert chunks(length=1 << 40) == nat.MI_ERR_UNSUPPORTED
    assert chunks(batch=0) == nat.MI_OK and chunks(length=0) == nat.MI_OK and chunks(width=-1) == nat.MI_ERR_INVALID

    def gather(batch=2, nb=3, stride=3, out=fine):
        return lib.mi_kv4_gather_blocks(fine, fine, fine, stride, None, 1, batch, nb, out, out, 8, 16, 8, 128, nat.MI_BF16,
                                        None)

    assert gather(stride=1) == nat.MI_ERR_INVALID
    assert gather(out=ctypes.c_void_p(264)) == nat.MI_ERR_INVALID and "16-byte" in nat.last_error()
    assert gather(batch=1 << 20, nb=1 << 20, stride=1 << 20) == nat.MI_ERR_UNSUPPORTED
    assert gather(batch=0) == nat.MI_OK and gather(nb=0) == nat.MI_OK

    def decode(batch=2, hq=16, width=4, stride=4, ws=None, ws_bytes=0, bs=16):
        return lib.mi_kv4_paged_decode(fine, s, None, None, None, None, fine, fine, 8, bs, 8, 128, fine, stride, width,
                                       fine, batch, hq, ctypes.c_float(1.0), fine, 0, ws, ws_bytes, nat.MI_BF16, None)

    assert decode(hq=12) == nat.MI_ERR_INVALID and "multiple" in nat.last_error()
    assert decode(width=0) == nat.MI_ERR_INVALID and decode(stride=3) == nat.MI_ERR_INVALID
    assert decode(batch=70000) == nat.MI_ERR_UNSUPPORTED and decode(batch=0) == nat.MI_OK
    assert decode(width=4096, stride=4096) == nat.MI_ERR_INVALID and "workspace" in nat.last_error()

    def append(slots=fine, d=128, bs=16, pool=fine):
        return lib.mi_kv4_qk_norm_rope(fine, 0, fine, 0, fine, 0, fine, fine, fine, fine, 0, 2, 16, 8, d, ctypes.c_float(1e-6),
                                       None, None, None, slots, pool, pool, 8, bs, nat.MI_BF16, None)

    assert append(slots=None) == nat.MI_ERR_INVALID and "slot_mapping" in nat.last_error()
    assert append(d=96) == nat.MI_ERR_UNSUPPORTED and append(bs=0) == nat.MI_ERR_INVALID
    assert append() == nat.MI_ERR_INVALID and "null pointer" in nat.last_error()  # q_out
    assert append(pool=None) == nat.MI_ERR_INVALID

    pools = (ctypes.c_void_p * 2)(256, None)
    assert lib.mi_kv_copy_blocks(pools, 2, fine, 3, 8, 64, None) == nat.MI_ERR_INVALID
    assert lib.mi_kv_copy_blocks(None, 2, fine, 3, 8, 64, None) == nat.MI_ERR_INVALID
    assert lib.mi_kv_copy_blocks(pools, 2, fine, 3, 0, 64, None) == nat.MI_ERR_INVALID
    assert lib.mi_kv_copy_blocks(pools, -1, fine, 3, 8, 64, None) == nat.MI_ERR_INVALID
    assert lib.mi_kv_copy_blocks(pools, 2, fine, 0, 8, 64, None) == nat.MI_OK
    assert lib.mi_kv_copy_blocks(pools, 0, None, 3, 8, 64, None) == nat.MI_OK


def test_workspace_is_bounded_and_host_only():
    lib = nat.load()
    size = lambda b, width: lib.mi_kv4_paged_decode_workspace_size(b, 32, 8, 128, width, 16, nat.MI_BF16)  # noqa: E731
    assert size(4, 8) == 0  # short tables: sequences are not cut
    assert 0 < size(1, 2048) <= size(512, 2048) == size(4096, 4096)  # two partials a persistent CTA at most
    assert lib.mi_kv4_paged_decode_workspace_size(4, 32, 8, 128, 2048, 16, nat.MI_F32) == 0


def test_oracle_write_and_read_are_inverse():
    rng = np.random.default_rng(0)
    pool = np.zeros((4, 2, ko.page_bytes(3, 96)), dtype=np.uint8)
    x = rng.standard_normal((5, 2, 96))
    x[0, 0, :32] = 1.25
    x[1, 1, 40] = np.inf
    slots = [1, 4, 5, 9, 2]
    ko.write(pool, x, slots, 3)
    got = ko.read(pool, range(4), 3, 96).reshape(12, 2, 96)
    assert np.array_equal(got[slots], ko.stored(x), equal_nan=True)
    assert np.isnan(got[4, 1, 32:64]).all() and (got[1, 0, :32] == 1.25).all()
    # half a step, the widest group's; its minimum and step are rounded to 8 bits
    ok = np.isfinite(x).reshape(5, 2, 3, 32).all(-1).repeat(32, -1)
    _, s, m = ko.quantise(x)
    bound = (s * (0.5 + 15 * 2.0**-8) + np.abs(m) * 2.0**-8).repeat(32, -1)
    assert (np.abs(got[slots] - x)[ok] <= bound[ok]).all()
