"""A 4-bit cache on a KV-head partition, host side (CPU, pools and exchange replaced by fakes): every rank's pool holds its
own heads, and its decode is followed by the process group's all-gather, not by the peer exchange."""

import pytest
import torch

from mini_infra_b200 import exchange
from mini_infra_b200.core import PagedCacheConfig, make_requests
from mini_infra_b200.engine import paged_schedule_backend as backend_mod
from mini_infra_b200.model import HeadPartition, Qwen3Config, build_model
from mini_infra_b200.model.config import TINY_C1


@pytest.mark.parametrize("kv_bits,kind", [(4, "PagedKV4CachePool"), (16, "PagedKVCachePool")])
@pytest.mark.parametrize("rank", [0, 1])
@pytest.mark.parametrize("peer_exchange", [True, False])
def test_pools_hold_local_heads_and_4_bits_take_the_all_gather(monkeypatch, kv_bits, kind, rank, peer_exchange):
    pools, attached = [], []

    class Pool:
        def __init__(self, **sizes):
            pools.append((self.name, sizes))
            self.kv_pools = []

    for name in ("PagedKV4CachePool", "PagedKVCachePool"):
        monkeypatch.setattr(backend_mod, name, type(name, (Pool,), {"name": name}))
    monkeypatch.setattr(exchange, "attach_peer_exchange", lambda *a: attached.append(a))
    cfg = Qwen3Config(**TINY_C1, torch_dtype="float32")
    model = build_model(cfg, seed=3, device="cpu", dtype=torch.float32, partition=HeadPartition(rank, 2, None))
    backend_mod.PagedScheduleBackend(model, make_requests([[1, 2, 3]], 4), 2, PagedCacheConfig(16, 8, kv_bits=kv_bits),
                                     cuda_graphs=False, peer_exchange=peer_exchange)
    (name, sizes), = pools
    assert name == kind and sizes["num_kv_heads"] == cfg.num_key_value_heads // 2 and sizes["head_dim"] == cfg.head_dim
    assert len(attached) == (kv_bits == 16 and peer_exchange)
