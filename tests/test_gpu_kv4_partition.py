"""A 4-bit cache on a KV-head partition, its two ranks one after the other on one GPU: what a rank's attention hands to
the all-gather, and what its pools hold, are the unpartitioned model's heads bit for bit (fp32: its kernels work head by head)."""

import pytest
import torch

from mini_infra_b200 import exchange, ops
from mini_infra_b200.core import PagedCacheConfig, make_requests
from mini_infra_b200.engine.paged_schedule_backend import PagedScheduleBackend
from mini_infra_b200.model import HeadPartition, Qwen3Config, build_model, qwen3
from mini_infra_b200.model.config import TINY_C1

pytestmark = pytest.mark.gpu
PROMPTS = [[(i * 37 + j * 11) % 900 + 1 for j in range(n)] for i, n in enumerate((5, 70, 33))]


def steps(model):
    """Two prefill chunks, three decode steps and a mixed one; the pools."""
    backend = PagedScheduleBackend(model, make_requests(PROMPTS, 12), 3, PagedCacheConfig(16, 32, kv_bits=4), cuda_graphs=False)
    m, runner, pool = backend.kv_cache_manager, backend.runner, backend.pool
    reqs, at = range(3), [0, 0, 0]
    for part in (0, 1):
        chunks = [p[: len(p) // 2] if part == 0 else p[len(p) // 2 :] for p in PROMPTS]
        for r in reqs:
            assert m.allocate_slots(r, len(chunks[r]))
        tables = [m.block_table(r) for r in reqs]
        out = runner.run_prefill_chunk_step(chunks, at, tables, pool)
        runner.store_prefill(pool, out.prefill_cache, tables, [len(c) for c in chunks], at)
        at = [a + len(c) for a, c in zip(at, chunks)]
    tokens = [3, 5, 7]
    for _ in range(3):
        for r in reqs:
            assert m.allocate_slots(r, 1)
        ids, pos, md = runner.prepare_decode_rows([(r, r) for r in reqs], [m.block_table(r) for r in reqs], tokens, at, 16)
        runner.run_decode_step(ids, pos, md, pool)
        tokens, at = [t + 1 for t in tokens], [a + 1 for a in at]
    for r in reqs:
        assert m.allocate_slots(r, 1)
    assert m.allocate_slots(3, 20)
    out = runner.run_mixed_step([m.block_table(r) for r in reqs], tokens, at, [list(range(1, 21))], [0], [m.block_table(3)], pool)
    runner.store_prefill(pool, out.prefill_cache, [m.block_table(3)], [20], [0])
    backend.close()
    return pool.kv_pools


@torch.inference_mode()
def test_the_ranks_heads_are_the_whole_models(monkeypatch):
    def never(*_):
        raise AssertionError("a 4-bit decode takes no peer exchange")

    monkeypatch.setattr(exchange, "attach_peer_exchange", never)
    tf32 = torch.backends.cuda.matmul.allow_tf32
    torch.backends.cuda.matmul.allow_tf32 = False
    cfg = Qwen3Config(**TINY_C1, torch_dtype="float32")
    build = lambda part: build_model(cfg, seed=5, device="cuda", dtype=torch.float32, partition=part)  # noqa: E731
    linear = qwen3._packed_linear
    attns, qkvs = [], []

    def record_attn(attn, partition):
        attns.append(attn.clone())
        return attn

    def record_qkv(x, weights, packed):
        got = linear(x, weights, packed)
        if len(weights) == 3:
            qkvs.append([t.clone() for t in got])
        return got

    monkeypatch.setattr(qwen3, "gather_heads", record_attn)
    monkeypatch.setattr(qwen3, "_packed_linear", record_qkv)
    whole = steps(build(HeadPartition()))
    assert len(attns) == len(qkvs) == 6 * cfg.num_hidden_layers
    for rank in (0, 1):
        attn_left, qkv_left = list(attns), list(qkvs)

        def rank_attn(attn, partition):
            every = attn_left.pop(0)
            width = every.shape[1] // 2
            assert torch.equal(attn, every[:, rank * width : (rank + 1) * width])
            return every  # what the all-gather gives every rank

        def rank_qkv(x, weights, packed):
            got = linear(x, weights, packed)
            if len(weights) != 3:
                return got
            mine = [t.chunk(2, dim=-1)[rank].contiguous() for t in qkv_left.pop(0)]
            for a, b in zip(got, mine):  # the same products; their order of sums is the library's
                assert a.shape == b.shape and torch.allclose(a, b, rtol=1e-3, atol=1e-4)
            return mine

        monkeypatch.setattr(qwen3, "gather_heads", rank_attn)
        monkeypatch.setattr(qwen3, "_packed_linear", rank_qkv)
        pools = steps(build(HeadPartition(rank, 2, None)))
        assert not attn_left and not qkv_left
        h = cfg.num_key_value_heads // 2
        for mine, every in zip(pools, whole):
            for a, b in zip(mine, every):
                assert torch.equal(a, b[:, rank * h : (rank + 1) * h])
    torch.backends.cuda.matmul.allow_tf32 = tf32
    assert ops.read_status() == 0
