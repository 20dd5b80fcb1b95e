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


def test_operands_of_other_types_and_shapes_are_refused():
    """Each would be read or written past its end, or as another type."""
    x = lambda dtype=torch.bfloat16, length=5, heads=2: torch.zeros((2, length, heads, 64), dtype=dtype)  # noqa: E731
    tables, lens = torch.zeros((2, 0), dtype=torch.long), torch.zeros(2, dtype=torch.long)
    for k, v, out in [(x(torch.half), x(torch.half), None), (x(), x(torch.float), None), (x(torch.float), x(), None),
                      (x(), x(length=4), None), (x(), x(heads=1), None),
                      (x(), x(), torch.zeros((2, 5, 256), dtype=torch.half))]:
        with pytest.raises(ValueError, match="alike"):
            ops.kv4_paged_prefill(x(heads=4), k, v, None, None, tables, lens, lens, 1.0, out=out)
    for q, k in [(x()[0], x()), (x(), x()[0])]:
        with pytest.raises(ValueError, match="heads, D"):
            ops.kv4_paged_prefill(q, k, k, None, None, tables, lens, lens, 1.0)
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        ops.kv4_paged_prefill(x(heads=4), x(), x(), None, None, tables, lens, lens, 1.0)
