"""The 4-bit cache as it is used: prompts stored and read back chunk by chunk, decode steps that append, forks
and compactions between them, the model and the engine on 4-bit pools."""

import numpy as np
import pytest
import torch

from mini_infra_b200 import ops
from mini_infra_b200.core import (
    BatchingMethod, ChunkedPrefillConfig, KVCacheManager, PagedCacheConfig, PrefillFirstConfig, SchedulerConfig,
    make_requests,
)
from mini_infra_b200.engine import EngineConfig, run_scheduler
from mini_infra_b200.model import PagedAttentionMetadata, Qwen3Config, build_model
from mini_infra_b200.model.config import TINY_C1
from mini_infra_b200.worker import PagedKV4CachePool, PagedKVCachePool, PagedRunner
from mini_infra_b200.worker.kv_cache import KVCache
from oracle import kv4_oracle as ko

pytestmark = pytest.mark.gpu


def np64(t):
    return t.detach().double().cpu().numpy()


def attention(q, k, v, scale):
    """One query [Hq, D] over k, v [n, H, D], in 64 bits."""
    g = q.shape[0] // k.shape[1]
    k, v = k.repeat(g, axis=1), v.repeat(g, axis=1)
    s = np.einsum("hd,thd->ht", q, k) * scale
    p = np.exp(s - s.max(-1, keepdims=True))
    return np.einsum("ht,thd->hd", p / p.sum(-1, keepdims=True), v).reshape(-1)


@pytest.mark.parametrize("dtype,d,hq,h,bs,close", [(torch.bfloat16, 128, 8, 4, 16, 2e-2), (torch.float32, 32, 4, 2, 3, 1e-4),
                                                   (torch.float16, 128, 8, 1, 32, 4e-3)])
def test_chunks_forks_compaction_and_decode_together(dtype, d, hq, h, bs, close):
    """Two prompts prefilled in two chunks each, one of them forked, the pool compacted, three decode steps:
    every output against 64-bit attention over what the cache stands for (the chunk's own K/V unquantised).
    Tolerance: the 16-bit prefill rounds keys, values and weights to its type, 2^-9 (bf16) or 2^-12 (fp16) of
    scores and values of a few units; 32 bits sum in another order."""
    g = torch.Generator(device="cuda").manual_seed(d)
    rnd = lambda *s: torch.randn(s, generator=g, device="cuda").to(dtype)  # noqa: E731
    m = KVCacheManager(bs, 40)
    pool = PagedKV4CachePool(2, 40, bs, h, d, dtype, torch.device("cuda"))
    scale = d**-0.5
    said = {r: ([], []) for r in range(3)}  # what the cache stands for, token by token, of layer 1
    m.allocate_slots(9, 2 * bs)  # a request that leaves, so that compaction has holes to fill
    tables_of = lambda reqs, width: torch.tensor([m.block_table(r)[:width] + [0] * (width - len(m.block_table(r)[:width]))  # noqa: E731
                                                  for r in reqs]).cuda()
    pos = {0: 0, 1: 0}
    for lens in ([5, 37], [40, 11]):
        reqs, width = [0, 1], max(lens)
        for r, n in zip(reqs, lens):
            assert m.allocate_slots(r, n)
        q, k, v = rnd(2, width, hq, d), rnd(2, width, h, d), rnd(2, width, h, d)
        starts = torch.tensor([pos[r] for r in reqs]).cuda()
        n_hist = max(-(-pos[r] // bs) for r in reqs)
        kp, vp = pool.kv_pools[1]
        out = ops.kv4_paged_prefill(q, k, v, kp, vp, tables_of(reqs, n_hist) if n_hist else torch.zeros((2, 0), dtype=torch.long).cuda(),
                                    starts, torch.tensor(lens).cuda(), scale)
        pool.store_chunks(KVCache([(k.transpose(1, 2), v.transpose(1, 2))] * 2), torch.tensor(lens).cuda(), starts,
                          tables_of(reqs, max(len(m.block_table(r)) for r in reqs)))
        for i, (r, n) in enumerate(zip(reqs, lens)):
            for j in range(n):
                at = width - n + j
                keys = np.array(said[r][0] + list(np64(k[i, width - n : at + 1]))).reshape(-1, h, d)
                vals = np.array(said[r][1] + list(np64(v[i, width - n : at + 1]))).reshape(-1, h, d)
                want = attention(np64(q[i, at]), keys, vals, scale)
                assert np.abs(np64(out[i, at]) - want).max() <= close
            for cache, x in zip(said[r], (k, v)):
                cache += list(ko.stored(np64(x[i, width - n :])))
            pos[r] += n
    m.free(9)
    moves = m.fork(1, 2)
    pool.copy_blocks(moves)
    said[2] = ([*said[1][0]], [*said[1][1]])
    pos[2] = pos[1]
    moves = m.compact()
    assert moves
    pool.copy_blocks(moves)
    for _ in range(3):
        reqs = [2, 0, 1]
        for r in reqs:
            assert m.allocate_slots(r, 1)
        q, k, v = rnd(3, hq, d), rnd(3, h, d), rnd(3, h, d)
        slots = torch.tensor([m.block_table(r)[pos[r] // bs] * bs + pos[r] % bs for r in reqs]).cuda()
        ctx = torch.tensor([pos[r] + 1 for r in reqs]).cuda()
        for kp, vp in pool.kv_pools:
            out = ops.kv4_paged_decode(q, kp, vp, tables_of(reqs, max(len(m.block_table(r)) for r in reqs)), ctx, scale,
                                       key_new=k, value_new=v, slot_mapping=slots)
        for i, r in enumerate(reqs):
            said[r][0].append(ko.stored(np64(k[i])))
            said[r][1].append(ko.stored(np64(v[i])))
            want = attention(np64(q[i]), np.array(said[r][0]), np.array(said[r][1]), scale)
            assert np.abs(np64(out[i]) - want).max() <= close
            pos[r] += 1
    assert ops.read_status() == 0


def test_pool_layout_byte_accounting_and_refusals():
    pool = PagedKV4CachePool(3, 10, 16, 2, 128, torch.bfloat16, torch.device("cuda"))
    kp, vp = pool.kv_pools[0]
    assert kp.shape == (10, 2, 1280) == vp.shape and not kp.any()
    assert pool.bytes_per_block == 2 * 3 * 2 * 1280 and pool.total_bytes == 10 * pool.bytes_per_block
    for pairs in ([(1, 10)], [(-1, 2)], [(1, 0)], [(1, 2), (3, 2)], [(1, 2), (2, 3)]):
        with pytest.raises(ValueError):
            pool.copy_blocks(pairs)
    pool.copy_blocks([])
    with pytest.raises(ValueError):
        PagedKV4CachePool(1, 4, 16, 2, 80, torch.bfloat16, torch.device("cuda"))
    with pytest.raises(RuntimeError):
        PagedKV4CachePool(1, 4, 16, 2, 128, torch.bfloat16, torch.device("cpu"))


@pytest.mark.parametrize("kind", [PagedKVCachePool, PagedKV4CachePool])
def test_copy_blocks_moves_every_layers_pages(kind):
    pool = kind(3, 8, 4, 2, 64, torch.bfloat16, torch.device("cuda"))
    for i, p in enumerate(x for layer in pool.kv_pools for x in layer):
        p.copy_(torch.randint(0, 100, p.shape, device="cuda") + i)
    before = [(k.clone(), v.clone()) for k, v in pool.kv_pools]
    pool.copy_blocks([(1, 5), (1, 6), (7, 2)])
    for (k, v), (k0, v0) in zip(pool.kv_pools, before):
        for now, old in ((k, k0), (v, v0)):
            old[5], old[6], old[2] = old[1].clone(), old[1].clone(), old[7].clone()
            assert torch.equal(now, old)


def model_of(dtype=torch.bfloat16, **more):
    cfg = Qwen3Config(**{**TINY_C1, "head_dim": 128, "hidden_size": 256, **more}, torch_dtype=str(dtype).split(".")[1])
    return build_model(cfg, seed=5, device="cuda", dtype=dtype)


@torch.inference_mode()
@pytest.mark.parametrize("dtype,head_dim,close", [(torch.bfloat16, 128, 3e-2), (torch.float32, 32, 1e-4)])
def test_decode_forward_equals_a_dense_pool_of_the_same_values(dtype, head_dim, close):
    """A decode forward on 4-bit pools against the same forward on dense pools that hold what the 4-bit ones
    stand for after the step's append: hidden states are normed rows of order one."""
    model = model_of(dtype, head_dim=head_dim)
    cfg, bs, nb = model.config, 16, 24
    g = torch.Generator(device="cuda").manual_seed(0)
    pool = PagedKV4CachePool(cfg.num_hidden_layers, nb, bs, cfg.num_key_value_heads, head_dim, dtype, torch.device("cuda"))
    shape = (1, cfg.num_key_value_heads, nb * bs, head_dim)
    fill = KVCache([tuple(torch.randn(shape, generator=g, device="cuda").to(dtype) for _ in range(2))
                    for _ in range(cfg.num_hidden_layers)])
    every = torch.arange(nb * bs).cuda()
    pool.write_prefill(fill, torch.zeros_like(every), every, every)
    ctx = torch.tensor([70, 33, 1]).cuda()
    tables = torch.tensor([[3, 7, 1, 9, 2], [4, 5, 6, 0, 0], [11, 0, 0, 0, 0]]).cuda()
    pos = ctx - 1
    slots = tables.gather(1, (pos // bs)[:, None])[:, 0] * bs + pos % bs
    ids = torch.randint(1, cfg.vocab_size, (3, 1), generator=g, device="cuda")
    md = PagedAttentionMetadata(slots, tables, ctx, tuple(pool.kv_pools))
    got, _ = model.model(ids, position_ids=pos[:, None], attn_metadata=md)
    dense = PagedKVCachePool(cfg.num_hidden_layers, nb, bs, cfg.num_key_value_heads, head_dim, dtype, torch.device("cuda"))
    values = pool.gather_blocks(torch.arange(nb).cuda()[None])
    for (kp, vp), (k, v) in zip(dense.kv_pools, values):
        kp.copy_(k[0].transpose(0, 1).view(kp.shape))
        vp.copy_(v[0].transpose(0, 1).view(vp.shape))
    # the dense forward would append its own unquantised token: write it to a slot of the null block instead
    want, _ = model.model(ids, position_ids=pos[:, None], attn_metadata=md._replace(
        slot_mapping=torch.arange(3).cuda(), kv_pools=tuple(dense.kv_pools)))
    assert (got - want).abs().max() <= close
    assert ops.read_status() == 0


PROMPTS = [[(i * 37 + j * 11) % 900 + 1 for j in range(n)] for i, n in enumerate((5, 70, 33, 150, 18))]


@pytest.mark.parametrize("dtype,head_dim", [(torch.bfloat16, 128), (torch.float32, 32)])
@pytest.mark.parametrize("policy", [PrefillFirstConfig(), ChunkedPrefillConfig(64), ChunkedPrefillConfig(64, mixed=True)],
                         ids=str)
def test_engine_runs_on_a_4bit_cache(policy, dtype, head_dim):
    """Graphs and eager steps give the same tokens; the pool is 3.2 (16 bits) or 6.4 times smaller."""
    model = model_of(dtype, head_dim=head_dim)
    ops.read_status()
    results = []
    for graphs in (True, False):
        cfg = EngineConfig(PagedCacheConfig(block_size=16, kv_bits=4), BatchingMethod.CONTINUOUS,
                           scheduler_config=SchedulerConfig(3, policy))
        results.append(run_scheduler(cfg, model, make_requests(PROMPTS, 12), None, stop_on_eos=False, cuda_graphs=graphs))
    assert [s.token_ids for s in results[0].sequences] == [s.token_ids for s in results[1].sequences]
    assert results[0].extra["decode_graph_replays"] + results[0].extra["mixed_graph_replays"] > 0
    assert all(s.output_len == 12 for s in results[0].sequences)
    assert ops.read_status() == 0
    full = run_scheduler(EngineConfig(PagedCacheConfig(block_size=16), BatchingMethod.CONTINUOUS,
                                      scheduler_config=SchedulerConfig(3, policy)), model, make_requests(PROMPTS, 12), None,
                         stop_on_eos=False)
    ratio = full.paged_cache.bytes_per_block / results[0].paged_cache.bytes_per_block
    assert ratio == pytest.approx(16 / 5 if dtype is torch.bfloat16 else 32 / 5)


@torch.inference_mode()
def test_compaction_between_decode_steps_changes_no_token():
    """Decode steps through the device's table mirror, the pool compacted in the middle of them."""
    from mini_infra_b200.engine.paged_schedule_backend import PagedScheduleBackend

    model = model_of()
    runs = []
    for compacted in (False, True):
        backend = PagedScheduleBackend(model, make_requests(PROMPTS, 12), 5, PagedCacheConfig(16, 64, kv_bits=4),
                                       cuda_graphs=False)
        m, runner, pool = backend.kv_cache_manager, backend.runner, backend.pool
        assert isinstance(runner, PagedRunner)
        for i, p in enumerate(PROMPTS):
            assert m.allocate_slots(i, len(p))
        out = runner.run_prefill_chunk_step(PROMPTS, [0] * 5, [m.block_table(i) for i in range(5)], pool)
        runner.store_prefill(pool, out.prefill_cache, [m.block_table(i) for i in range(5)], [len(p) for p in PROMPTS],
                             [0] * 5)
        m.free(1)  # leaves holes
        live, tokens, pos = [0, 2, 3, 4], dict(enumerate(out.next_tokens)), {i: len(p) for i, p in enumerate(PROMPTS)}
        seen = []
        for step in range(8):
            if compacted and step in (2, 5):
                assert (backend.compact() > 0) == (step == 2)
            for i in live:
                assert m.allocate_slots(i, 1)
            ids, ps, md = runner.prepare_decode_rows([(i, i) for i in live], [m.block_table(i) for i in live],
                                                     [tokens[i] for i in live], [pos[i] for i in live], 16)
            for i, t in zip(live, runner.run_decode_step(ids, ps, md, pool).next_tokens):
                tokens[i], pos[i] = t, pos[i] + 1
                seen.append(t)
        runs.append(seen)
        backend.close()
    assert runs[0] == runs[1]
    assert ops.read_status() == 0
