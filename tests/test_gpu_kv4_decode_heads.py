"""Decodes with four KV heads a CTA and up to eight query heads each, in blocks of 16 and 32 (those of large models),
against the oracle, within the tolerance of the other decodes."""

import numpy as np
import pytest
import torch

from mini_infra_b200 import ops
from oracle import kv4_oracle as ko
from test_gpu_kv4 import cuda, decode_case, decode_tolerance, np64, pools, tokens

pytestmark = pytest.mark.gpu

HEADS = [
    # query heads, KV heads, head_dim, block size
    (64, 8, 128, 16), (40, 8, 128, 16), (20, 4, 64, 16), (28, 4, 64, 32), (16, 4, 128, 32), (32, 4, 128, 32), (24, 4, 128, 32),
    (4, 4, 64, 32), (16, 2, 128, 16), (10, 2, 64, 32), (8, 1, 128, 32), (5, 1, 64, 16), (6, 1, 128, 16), (7, 1, 64, 32),
]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("hq,h,d,bs", HEADS)
def test_short_and_middling_rows(hq, h, d, bs, dtype):
    scale = d**-0.5
    for lengths in ((1, 2 * bs + 1), (1, 700)):
        q, kp, vp, tables, ctx = decode_case(4, hq, h, d, bs, lengths, dtype)
        got = ops.kv4_paged_decode(q, cuda(kp), cuda(vp), cuda(tables), cuda(ctx), scale)
        assert ops.read_status() == 0
        want = ko.decode(np64(q), kp, vp, tables, ctx, scale, bs)
        err = np.abs(np64(got) - want)
        tol = decode_tolerance(want, np64(q), kp, vp, tables, ctx, scale, bs, dtype)
        assert (err <= tol).all(), f"{(err / tol).max():.2f} of the tolerance"


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("b,longest", [(60, 1500), (3, 6001)])
@pytest.mark.parametrize("hq,h,d,bs", HEADS)
def test_cut_rows_among_empty_ones(hq, h, d, bs, b, longest, dtype):
    """Rows cut over CTAs, pages poisoned past every length, rows of no tokens at both ends and between."""
    rng = np.random.default_rng(hq + b)
    ctx = np.minimum(rng.geometric(4 / longest, b), longest).astype(np.int64)
    ctx[1] = longest
    ctx[[0, -1]] = 0
    ctx[rng.integers(2, b, b // 8)] = 0
    # full pages are shared by the rows; the last page of each is its own, with NaN parameters past the length
    shared = 48
    kp, vp = pools(rng, shared, bs, h, d)
    own = np.full((b, *kp.shape[1:]), 0xFF, dtype=np.uint8)
    kp, vp = np.concatenate((kp, own)), np.concatenate((vp, own))
    tables = rng.integers(1, shared, (b, -(-longest // bs) + 1)).astype(np.int64)
    for i, n in enumerate(ctx):
        if n:
            last, left = (n - 1) // bs, int((n - 1) % bs + 1)
            tables[i, last] = shared + i
            for pool in (kp, vp):
                ko.write(pool, np64(tokens(rng, (left, h, d), "bf16")), [(shared + i) * bs + t for t in range(left)], bs)
    q = tokens(rng, (b, hq, d), dtype)
    scale = d**-0.5
    got = ops.kv4_paged_decode(q, cuda(kp), cuda(vp), cuda(tables), cuda(ctx), scale)
    assert ops.read_status() == 0
    want = ko.decode(np64(q), kp, vp, tables, ctx, scale, bs)
    tol = decode_tolerance(want, np64(q), kp, vp, tables, ctx, scale, bs, dtype)
    err = np.abs(np64(got) - want)
    assert (err <= tol).all(), f"{(err / tol).max():.2f} of the tolerance"
    assert not got[torch.from_numpy(ctx == 0).cuda()].any()
    assert torch.equal(got, ops.kv4_paged_decode(q, cuda(kp), cuda(vp), cuda(tables), cuda(ctx), scale))
