"""Decode over long flat rows of the 4-bit cache: the output is hundreds of times smaller than the weighted codes and
minima that it is the sum of, so that what a long sum loses shows."""

import numpy as np
import pytest
import torch

from mini_infra_b200 import ops
from oracle import kv4_oracle as ko

pytestmark = pytest.mark.gpu
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}

CASES = [
    # rows, query heads, KV heads, head_dim, block size, tokens, dtype; with 450 rows and more a warp takes whole rows
    (900, 4, 4, 128, 16, 32768, "fp16"),
    (900, 4, 4, 128, 16, 32768, "bf16"),
    (900, 8, 1, 128, 32, 32768, "fp16"),  # a quarter of a row a warp
    (600, 12, 6, 64, 16, 16384, "bf16"),
    (600, 12, 6, 64, 32, 16384, "fp16"),
    (450, 32, 4, 128, 16, 8192, "fp16"),
    (450, 20, 4, 128, 32, 8192, "bf16"),
    (1, 8, 1, 128, 32, 32768, "fp16"),    # one row over many CTAs
]


def sums_tolerance(q, k, v_pool, ids, want, n, scale, bs, dtype):
    """A bound on |decode - exact| of one row, [Hq, D], for independent roundings: those of n terms add as the root
    of their squares, six standard deviations of it.

    * the output's rounding: half a unit, 2^-25 below fp16's normal range;
    * p s in fp16: each off by at most 2^-11 of it, 2^-11 / sqrt(3) as a standard deviation, times at most 8 steps (the
      codes count from their middle); fp16 models carry the rest, whose products lose at most 2^-20 of a step;
    * sums in fp32, one rounding of 2^-24 an addition: O, 16 tokens at a time, of partial sums that reach about
      3 * 8 sqrt(sum (p s)^2); the middles m + 8 s and the weights, a token in eight at a time, of partial sums of
      at most sum p |m + 8 s| and 1;
    * the weights: a score is a sum of 2 D terms within 2^-24 each, the exponential within 2^-21; twice that of
      sum p |v|.
    """
    hq, d = q.shape
    h = v_pool.shape[1]
    rep = lambda x: x.repeat(hq // h, axis=0)  # noqa: E731
    x = np.einsum("hd,thd->ht", q, k.repeat(hq // h, axis=1)) * scale
    p = np.exp(x - x.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    ng = d // ko.GROUP
    par = np.ascontiguousarray(v_pool[ids][..., ng * bs * 16 :]).view("<u2").reshape(-1, h, bs, ng, 2)
    par = (par.transpose(0, 2, 1, 3, 4).reshape(-1, h, ng, 2)[:n].astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    step, mid = par[..., 0].transpose(1, 0, 2), par[..., 1].transpose(1, 0, 2) + 8 * par[..., 0].transpose(1, 0, 2)
    step, mid = rep(step), rep(mid)  # [Hq, n, groups]
    root = np.sqrt(np.einsum("ht,htg->hg", p**2, step**2))
    weighted = 2.0**-11 / np.sqrt(3) * 8 * root * 6 if dtype == "bf16" else 2.0**-20 * np.einsum("ht,htg->hg", p, step)
    sums = 6 * np.sqrt(n / 16) * 2.0**-24 * 24 * root + 6 * np.sqrt(n / 8) * 2.0**-24 * np.einsum("ht,htg->hg", p, np.abs(mid))
    delta = (2 * d + 64) * 2.0**-24 * scale * np.einsum("hd,thd->ht", np.abs(q), np.abs(k).repeat(hq // h, axis=1)).max(-1)
    size = np.einsum("ht,htg->hg", p, np.maximum(np.abs(mid - 8 * step), np.abs(mid + 7 * step)))
    tol = weighted + sums + 2 * (np.expm1(delta) + 2.0**-21)[:, None] * size
    half = torch.finfo(DTYPES[dtype]).eps / 2
    return (tol.repeat(ko.GROUP, axis=1) + (half + 6 * np.sqrt(n / 8) * 2.0**-24) * np.abs(want) * 1.01
            + (2.0**-25 if dtype == "fp16" else 1e-30))


def long_rows(b, hq, h, d, bs, n, dtype, spread):
    """(query, pools, tables): rows over the same pages, each in an order of its own."""
    g = torch.Generator(device="cuda").manual_seed(b + hq + d)
    rnd = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    pages = n // bs
    kp = torch.zeros((pages + 1, h, ops.kv4_page_bytes(bs, d)), dtype=torch.uint8, device="cuda")
    vp = torch.zeros_like(kp)
    ops.kv4_scatter(rnd(n, h, d).to(DTYPES[dtype]), rnd(n, h, d).to(DTYPES[dtype]), None, None,
                    torch.arange(bs, bs + n).cuda(), kp, vp)
    tables = 1 + torch.rand((b, pages), generator=g, device="cuda").argsort(dim=1)
    return (spread * rnd(b, hq, d)).to(DTYPES[dtype]), kp, vp, tables


@pytest.mark.parametrize("b,hq,h,d,bs,n,dtype", CASES)
def test_long_flat_rows_keep_their_small_outputs(b, hq, h, d, bs, n, dtype):
    q, kp, vp, tables = long_rows(b, hq, h, d, bs, n, dtype, 0.05)
    scale = d**-0.5
    got = ops.kv4_paged_decode(q, kp, vp, tables, torch.full((b,), n).cuda(), scale)
    assert ops.read_status() == 0
    kp, vp = kp.cpu().numpy(), vp.cpu().numpy()
    for i in sorted({0, b // 2, b - 1}):
        ids = tables[i].cpu().numpy()
        qi = q[i].double().cpu().numpy()
        want = ko.decode(qi[None], kp, vp, ids[None], [n], scale, bs).reshape(hq, d)
        k = ko.read(kp, ids, bs, d).reshape(-1, h, d)
        tol = sums_tolerance(qi, k, vp, ids, want, n, scale, bs, dtype)
        err = np.abs(got[i].double().cpu().numpy().reshape(hq, d) - want)
        assert (err <= tol).all(), f"row {i}: {(err / tol).max():.2f} of the tolerance"


@pytest.mark.parametrize("b,dtype", [(8, "fp16"), (8, "bf16"), (500, "fp16"), (500, "bf16")])
def test_long_rows_of_unlike_weights_have_no_bias(b, dtype):
    """The mean error of N outputs whose roundings are independent, each of a standard deviation of at most half a unit
    / sqrt(3) of its output (bf16: and a quarter of that for the weights' own): six standard deviations of the mean."""
    hq, h, d, bs, n = 8, 1, 128, 32, 32768
    q, kp, vp, tables = long_rows(b, hq, h, d, bs, n, dtype, 1.0)
    got = ops.kv4_paged_decode(q, kp, vp, tables, torch.full((b,), n).cuda(), d**-0.5)
    kp, vp = kp.cpu().numpy(), vp.cpu().numpy()
    rows = list(range(8)) if b == 8 else [0, 100, 200, 300, 400, 499]
    want = np.stack([ko.decode(q[i : i + 1].double().cpu().numpy(), kp, vp, tables[i : i + 1].cpu().numpy(), [n], d**-0.5, bs)[0]
                     for i in rows])
    error = (got[rows].double().cpu().numpy() - want).mean() / np.sqrt((want**2).mean())
    half = torch.finfo(DTYPES[dtype]).eps / 2
    assert abs(error) <= 6 * 1.04 * half / np.sqrt(3) / np.sqrt(want.size)
