"""Prefill and mixed step graphs over a 4-bit pool: what they keep on the device, and their tokens against eager
steps over histories of every bucket."""

import pytest
import torch

from mini_infra_b200 import ops
from mini_infra_b200.core import (
    BatchingMethod, ChunkedPrefillConfig, PagedCacheConfig, SchedulerConfig, make_requests,
)
from mini_infra_b200.engine import EngineConfig, run_scheduler
from mini_infra_b200.model import Qwen3Config, build_model
from mini_infra_b200.model.config import TINY_C1
from mini_infra_b200.worker import PagedKV4CachePool, PagedRunner

pytestmark = pytest.mark.gpu


def model_of(dtype, head_dim):
    cfg = Qwen3Config(**{**TINY_C1, "head_dim": head_dim, "hidden_size": 256}, torch_dtype=str(dtype).split(".")[1])
    return build_model(cfg, seed=5, device="cuda", dtype=dtype)


@torch.inference_mode()
def test_a_captured_step_without_history_keeps_no_dense_history():
    """Tables of 2,048 blocks; a dense copy of 16 rows of them takes 537 MB.  What else a step of 16 chunks of 32
    tokens takes: the MLP's and attention's rows, the logits, and the prefill's workspace (some 39 MB)."""
    model = model_of(torch.bfloat16, 128)
    cfg, bs, width, rows = model.config, 16, 2048, 16
    pool = PagedKV4CachePool(cfg.num_hidden_layers, 64, bs, cfg.num_key_value_heads, 128, torch.bfloat16, torch.device("cuda"))
    dense = 2 * rows * width * bs * cfg.num_key_value_heads * 128 * 2
    runner = PagedRunner(model, 0)
    runner.enable_mixed_graphs(pool, width)
    chunks = [[(7 * i + j) % 900 + 1 for j in range(30)] for i in range(rows)]
    tables = [[2 * i + 1, 2 * i + 2] for i in range(rows)]
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_reserved()
    assert runner.warm_mixed_graph([], chunks, tables, pool, [0] * rows)
    got = runner.run_mixed_step([], [], [], chunks, [0] * rows, tables, pool)
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_reserved() - before < dense // 2
    want = runner.run_prefill_chunk_step(chunks, [0] * rows, tables, pool)
    assert got.prefill_tokens == want.next_tokens
    # with history: a copy of the bucket's columns, not of the table's
    more = [[t + 1 for t in c[:2]] for c in chunks]
    assert runner.warm_mixed_graph([], more, tables, pool, [30] * rows)
    got = runner.run_mixed_step([], [], [], more, [30] * rows, tables, pool)
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_reserved() - before < dense // 2
    want = runner.run_prefill_chunk_step(more, [30] * rows, tables, pool)
    assert got.prefill_tokens == want.next_tokens
    assert runner.prefill_graph_replays == 2 and ops.read_status() == 0
    runner.release_mixed_graphs()


@pytest.mark.parametrize("dtype,head_dim,bs", [(torch.bfloat16, 128, 16), (torch.float32, 32, 1)])
@pytest.mark.parametrize("mixed", [False, True])
def test_histories_of_every_bucket_give_the_eager_tokens(dtype, head_dim, bs, mixed):
    """Prompts prefilled in chunks, so that histories pass through the buckets (blocks of one token: up to 1,024)."""
    model = model_of(dtype, head_dim)
    prompts = [[(i * 37 + j * 11) % 900 + 1 for j in range(n)] for i, n in enumerate((400, 30, 170))]
    ops.read_status()
    runs = []
    for graphs in (True, False):
        cfg = EngineConfig(PagedCacheConfig(block_size=bs, kv_bits=4), BatchingMethod.CONTINUOUS,
                           scheduler_config=SchedulerConfig(3, ChunkedPrefillConfig(64, mixed=mixed)))
        runs.append(run_scheduler(cfg, model, make_requests(prompts, 6), None, stop_on_eos=False, cuda_graphs=graphs))
    assert [s.token_ids for s in runs[0].sequences] == [s.token_ids for s in runs[1].sequences]
    assert runs[0].extra["prefill_graph_replays"] + runs[0].extra["mixed_graph_replays"] > 3
    assert ops.read_status() == 0
