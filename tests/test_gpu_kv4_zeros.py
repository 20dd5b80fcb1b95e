"""Groups whose smallest value is a zero of either sign: the store, the chunk store and the append fused with norm
and RoPE leave the same bytes, the oracle's."""

import numpy as np
import pytest
import torch

from mini_infra_b200 import ops
from oracle import kv4_oracle as ko

pytestmark = pytest.mark.gpu
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def signed_zeros(rng, t, h, d, dtype):
    """Groups of -0 alone, of both zeros, of non-negative values with a -0 (or both) among them, of tiny negative
    values that bfloat16 rounds to -0 (fp32), and ordinary ones."""
    x = rng.standard_normal((t, h, d // 32, 32)).astype(np.float32)
    kind = rng.integers(0, 6, x.shape[:-1])
    kind.reshape(-1)[:6] = range(6)
    minus = np.float32(-0.0)
    x[kind == 0] = minus
    x[kind == 1] = np.where(rng.random(x[kind == 1].shape) < 0.5, minus, np.float32(0))
    for k in (2, 3):
        x[kind == k] = np.abs(x[kind == k])
    x[kind == 2, rng.integers(32)] = minus
    x[kind == 3, :2] = [0.0, minus]
    x[kind == 4] = np.float32(-1e-45)
    return torch.from_numpy(x.reshape(t, h, d)).to(DTYPES[dtype]).cuda()


@pytest.mark.parametrize("d", [32, 64, 128, 256])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_zero_minima_have_no_sign(d, dtype):
    rng = np.random.default_rng(d)
    t, h, bs, n = 24, 2, 8, 4
    k, v = signed_zeros(rng, t, h, d, dtype), signed_zeros(rng, t, h, d, dtype)
    new = lambda: [torch.zeros((n, h, ops.kv4_page_bytes(bs, d)), dtype=torch.uint8, device="cuda") for _ in range(2)]  # noqa: E731
    slots = torch.arange(bs, bs + t).cuda()
    stored, chunks, fused = new(), new(), new()
    ops.kv4_scatter(k, v, None, None, slots, *stored)
    ops.kv4_store_chunks(k.transpose(0, 1)[None], v.transpose(0, 1)[None], torch.tensor([t]).cuda(), torch.tensor([0]).cuda(),
                         torch.tensor([[1, 2, 3]]).cuda(), *chunks)
    for pool, other, x in zip(stored, chunks, (k, v)):
        want = np.zeros(tuple(pool.shape), dtype=np.uint8)
        ko.write(want, x.double().cpu().numpy(), range(bs, bs + t), bs)
        assert np.array_equal(pool.cpu().numpy(), want)
        assert torch.equal(pool, other)
    # the fused append against the store of its own outputs: V as it is, K's zeros through norm and RoPE
    q = torch.zeros((t, h * d), dtype=k.dtype, device="cuda")
    weight = torch.ones(d, dtype=k.dtype, device="cuda")
    cos, sin = torch.ones((t, d), dtype=k.dtype, device="cuda"), torch.zeros((t, d), dtype=k.dtype, device="cuda")
    args = (q, k.reshape(t, -1), v.reshape(t, -1), weight, weight, cos, sin, 1e-6, h, h)
    ops.kv4_qk_norm_rope(*args, slots, *fused)
    _, k_out, v_out = ops.qk_norm_rope(*args)
    apart = new()
    ops.kv4_scatter(k_out, v_out, None, None, slots, *apart)
    assert torch.equal(fused[0], apart[0]) and torch.equal(fused[1], apart[1])
    assert torch.equal(fused[1], stored[1])
    assert ops.read_status() == 0
