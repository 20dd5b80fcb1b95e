"""Host side of the prefill over a 4-bit history: which device is current when it launches (CPU, with a fake of the
calls below it)."""

from types import SimpleNamespace

import pytest
import torch

from mini_infra_b200 import _native as nat
from mini_infra_b200 import ops


class FakeCuda:
    """Two devices, the first of them current."""

    def __init__(self):
        self.current = 0

    def device(self, device):
        fake = self

        class Guard:
            def __enter__(self):
                self.before, fake.current = fake.current, device.index

            def __exit__(self, *_):
                fake.current = self.before

        return Guard()


@pytest.mark.parametrize("index", [0, 1])
@pytest.mark.parametrize("blocks", [0, 2])
def test_it_launches_with_its_tensors_device_current(monkeypatch, index, blocks):
    cuda, seen = FakeCuda(), []
    monkeypatch.setattr(torch.cuda, "current_device", lambda: cuda.current)
    monkeypatch.setattr(torch.cuda, "device", cuda.device)
    meta = lambda *s, **k: torch.empty(s, device="meta", **k)  # noqa: E731

    def fake_gather(kp, vp, ids, d, dtype, lengths, fill_past):
        seen.append(cuda.current)
        return meta(2, blocks, 16, 2, d, dtype=dtype), meta(2, blocks, 16, 2, d, dtype=dtype)

    def fake_prefill(query, *args, **kwargs):
        seen.append(cuda.current)
        return "out"

    monkeypatch.setattr(ops, "kv4_gather_blocks", fake_gather)
    monkeypatch.setattr(ops, "paged_prefill", fake_prefill)
    monkeypatch.setattr(nat, "load", lambda: SimpleNamespace(mi_paged_prefill_workspace_size=lambda *a: 0))
    for name in ("arange", "empty"):
        real = getattr(torch, name)
        monkeypatch.setattr(torch, name, lambda *a, _real=real, **k: _real(*a, **{**k, "device": "meta"}))
    query = SimpleNamespace(ndim=4, shape=(2, 5, 4, 64), dtype=torch.bfloat16, device=torch.device("cuda", index))
    chunk = SimpleNamespace(ndim=4, shape=(2, 5, 2, 64), dtype=torch.bfloat16, device=query.device)
    tables = meta(2, blocks, dtype=torch.long)
    lens = meta(2, dtype=torch.long)
    assert ops.kv4_paged_prefill(query, chunk, chunk, None, None, tables, lens, lens, 1.0) == "out"
    assert seen == [index] * (1 + (blocks > 0)) and cuda.current == 0
