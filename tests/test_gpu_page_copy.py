"""Block copies inside every pool of a cache (mi_kv_copy_blocks): bit for bit, nothing else touched."""

import pytest
import torch

from mini_infra_b200 import _native as nat
from mini_infra_b200 import ops

pytestmark = pytest.mark.gpu


def make(shape, dtype, count, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randint(0, 256, (torch.empty(shape, dtype=dtype).nbytes,), generator=g, device="cuda",
                          dtype=torch.uint8).view(dtype).view(shape) for _ in range(count)]


@pytest.mark.parametrize("shape,dtype", [((9, 16, 8, 128), torch.bfloat16), ((9, 3, 1, 32), torch.float32),
                                         ((9, 1, 1, 3), torch.float16), ((9, 2, 1280), torch.uint8),
                                         ((9, 1, 20), torch.uint8), ((9, 7), torch.uint8)])
@pytest.mark.parametrize("count", [1, 2, 56, 300])
def test_copies_are_exact_in_every_pool(shape, dtype, count):
    pools = make(shape, dtype, count)
    before = [p.view(torch.uint8).clone() for p in pools]
    ops.kv_copy_blocks(pools, torch.tensor([[1, 4], [1, 5], [8, 2], [3, 3]]).cuda())
    assert ops.read_status() == 0
    for p, old in zip(pools, before):
        old[4], old[5], old[2] = old[1].clone(), old[1].clone(), old[8].clone()
        assert torch.equal(p.view(torch.uint8), old)


def test_misaligned_pools():
    base = torch.randint(0, 256, (1 + 9 * 48,), dtype=torch.uint8, device="cuda")
    pool = base[1:].view(9, 48)
    want = pool.clone()
    want[7] = want[2]
    ops.kv_copy_blocks([pool], torch.tensor([[2, 7]]).cuda())
    assert torch.equal(pool, want)


def test_bad_ids_are_flagged_and_skipped():
    pools = make((4, 2, 32), torch.bfloat16, 3)
    before = [p.view(torch.uint8).clone() for p in pools]
    ops.read_status()
    ops.kv_copy_blocks(pools, torch.tensor([[1, 4], [-1, 2], [4, 1], [1 << 40, 3]]).cuda())
    assert ops.read_status() == nat.MI_STATUS_BAD_BLOCK
    assert all(torch.equal(p.view(torch.uint8), o) for p, o in zip(pools, before))


def test_a_captured_copy_follows_its_pairs():
    pools = make((6, 4, 64), torch.float16, 4)
    pairs = torch.tensor([[1, 2], [0, 0]]).cuda()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.kv_copy_blocks(pools, pairs)
    pairs.copy_(torch.tensor([[3, 4], [1, 5]]))
    g.replay()
    torch.cuda.synchronize()
    for p in pools:
        p = p.view(torch.uint8)
        assert torch.equal(p[4], p[3]) and torch.equal(p[5], p[1]) and not torch.equal(p[2], p[1])


def test_refusals():
    a, b = make((4, 2, 32), torch.bfloat16, 2)
    pairs = torch.tensor([[1, 2]]).cuda()
    for args in [([a, b[:3]], pairs), ([a, b.float()], pairs), ([a.transpose(1, 2)], pairs), ([a], pairs.int()),
                 ([a], pairs.view(-1)), ([a], torch.zeros((2, 3), dtype=torch.long).cuda()), ([a.view(-1)], pairs)]:
        with pytest.raises(ValueError):
            ops.kv_copy_blocks(*args)
    with pytest.raises(RuntimeError):
        ops.kv_copy_blocks([a.cpu()], pairs)
    ops.kv_copy_blocks([], pairs)
    ops.kv_copy_blocks([a], pairs[:0])
    ops.kv_copy_blocks([a[:0]], pairs)
