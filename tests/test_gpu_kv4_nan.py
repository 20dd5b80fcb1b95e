"""A token whose key the cache holds as NaN makes every output that attends to it NaN, wherever it stands, and no
other output: decodes on the tensor-core shapes and on the others, against the clean pool's and the definition."""

import numpy as np
import pytest
import torch

from mini_infra_b200 import ops
from oracle import kv4_oracle as ko

pytestmark = pytest.mark.gpu
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SHAPES = [
    # query heads, KV heads, head_dim, block size, dtype
    (4, 2, 32, 4, "fp32"), (32, 2, 128, 16, "bf16"), (6, 3, 96, 16, "fp16"), (2, 2, 256, 5, "fp32"), (4, 2, 128, 8, "bf16"),
    (8, 4, 128, 16, "bf16"), (16, 2, 64, 32, "fp16"),  # tensor cores
]


@pytest.mark.parametrize("where", ["first", "later_page", "first_of_every_page", "all", "last"])
@pytest.mark.parametrize("hq,h,d,bs,dtype", SHAPES)
def test_a_nan_key_spoils_its_heads_row_wherever_it_stands(hq, h, d, bs, dtype, where):
    rng = np.random.default_rng(d)
    n = 11 * bs + 1
    rows = 3
    pages = -(-n // bs)
    tables = (1 + rng.permutation(rows * pages)).reshape(rows, pages).astype(np.int64)
    pools = []
    for _ in range(2):
        pool = np.zeros((rows * pages + 1, h, ko.page_bytes(bs, d)), dtype=np.uint8)
        ko.write(pool, rng.standard_normal((pool.shape[0] * bs, h, d)), range(pool.shape[0] * bs), bs)
        pools.append(pool)
    spoiled = {"first": [0], "later_page": [9 * bs], "first_of_every_page": range(0, n, bs), "all": range(n),
               "last": [n - 1]}[where]
    kp = torch.from_numpy(pools[0]).cuda()
    vp = torch.from_numpy(pools[1]).cuda()
    tab, ctx = torch.from_numpy(tables).cuda(), torch.full((rows,), n).cuda()
    q = torch.from_numpy(rng.standard_normal((rows, hq, d))).to(DTYPES[dtype]).cuda()
    clean = ops.kv4_paged_decode(q, kp, vp, tab, ctx, 0.1).view(rows, h, -1, d)
    assert torch.isfinite(clean).all()
    groups = kp[..., d // 32 * bs * 16 :].view(torch.bfloat16).view(-1, h, bs, d // 32, 2)
    for t in spoiled:  # as a store leaves a group that held a NaN: step 0, minimum NaN
        groups[tables[1, t // bs], h - 1, t % bs, 0] = torch.tensor([0.0, float("nan")], dtype=torch.bfloat16)
    got = ops.kv4_paged_decode(q, kp, vp, tab, ctx, 0.1).view(rows, h, -1, d)
    assert torch.isnan(got[1, h - 1]).all()
    got[1, h - 1] = clean[1, h - 1]
    assert torch.equal(got, clean)
    assert ops.read_status() == 0


@pytest.mark.parametrize("hq,h,d,bs,dtype", SHAPES)
def test_a_nan_value_spoils_its_group_alone(hq, h, d, bs, dtype):
    rng = np.random.default_rng(d + 1)
    n = 3 * bs
    pool = np.zeros((4, h, ko.page_bytes(bs, d)), dtype=np.uint8)
    ko.write(pool, rng.standard_normal((4 * bs, h, d)), range(4 * bs), bs)
    kp = torch.from_numpy(pool).cuda()
    vp = kp.clone()
    q = torch.from_numpy(rng.standard_normal((1, hq, d))).to(DTYPES[dtype]).cuda()
    tab, ctx = torch.tensor([[3, 1, 2]]).cuda(), torch.tensor([n]).cuda()
    clean = ops.kv4_paged_decode(q, kp, vp, tab, ctx, 0.1).view(h, -1, d // 32, 32)
    vp[..., d // 32 * bs * 16 :].view(torch.bfloat16).view(-1, h, bs, d // 32, 2)[3, 0, 0, 0] = torch.tensor(
        [0.0, float("nan")], dtype=torch.bfloat16)
    got = ops.kv4_paged_decode(q, kp, vp, tab, ctx, 0.1).view(h, -1, d // 32, 32)
    assert torch.isnan(got[0, :, 0]).all()
    got[0, :, 0] = clean[0, :, 0]
    assert torch.equal(got, clean)
