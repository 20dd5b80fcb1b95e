"""The 4-bit paged cache on the GPU: store, gather and decode against the oracle in 64 bits.

What a store leaves in a page is compared byte for byte with the oracle (16-bit sources: every step of
the quantiser is exact or rounded once in both), a gather bit for bit, a decode within a tolerance
summed from its roundings (``decode_tolerance``).
"""

import numpy as np
import pytest
import torch

from mini_infra_b200 import _native as nat
from mini_infra_b200 import ops
from oracle import kv4_oracle as ko

pytestmark = pytest.mark.gpu
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


@pytest.fixture(autouse=True)
def clean_status():
    ops.read_status()
    yield
    torch.cuda.synchronize()


def tokens(rng, shape, dtype):
    """Values with a mean and a width of their own per channel, some groups constant, some tiny."""
    x = rng.standard_normal(shape) * (0.2 + rng.random(shape[-1])) + rng.standard_normal(shape[-1])
    x = x.reshape(-1, ko.GROUP)
    x[rng.integers(0, len(x), max(1, len(x) // 16))] = 0.75
    x[rng.integers(0, len(x), max(1, len(x) // 16))] *= 1e-3
    return torch.from_numpy(x.reshape(shape)).to(DTYPES[dtype]).cuda()


def np64(t):
    return t.detach().double().cpu().numpy()


def pools(rng, blocks, bs, h, d):
    """Pools quantised from random tokens, as numpy (the oracle's own bytes)."""
    got = []
    for _ in range(2):
        pool = np.zeros((blocks, h, ko.page_bytes(bs, d)), dtype=np.uint8)
        x = np64(tokens(rng, (blocks * bs, h, d), "bf16"))
        ko.write(pool, x, range(blocks * bs), bs)
        got.append(pool)
    return got


def cuda(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def tables_for(rng, lengths, bs, extra=1):
    need = [-(-int(n) // bs) for n in lengths]
    blocks = 1 + sum(need) + 3
    ids = list(1 + rng.permutation(blocks - 1))
    tables = np.zeros((len(need), max(need) + extra), dtype=np.int64)
    for i, n in enumerate(need):
        tables[i, :n] = [ids.pop() for _ in range(n)]
    return tables, blocks


# ---------------------------------------------------------------------------------------------
# store
# ---------------------------------------------------------------------------------------------
STORE = [
    # batch, heads, head_dim, block size, dtype
    (5, 8, 128, 16, "bf16"), (3, 2, 64, 16, "fp16"), (4, 1, 32, 3, "bf16"), (2, 3, 96, 1, "fp16"),
    (7, 4, 256, 32, "bf16"), (1, 5, 160, 4, "bf16"),
]


@pytest.mark.parametrize("b,h,d,bs,dtype", STORE)
def test_append_writes_the_oracles_bytes(b, h, d, bs, dtype):
    rng = np.random.default_rng(b * 100 + d)
    blocks = b + 3
    want = pools(rng, blocks, bs, h, d)
    kp, vp = cuda(want[0]), cuda(want[1])
    k, v = tokens(rng, (b, h, d), dtype), tokens(rng, (b, h, d), dtype)
    slots = rng.permutation(blocks * bs)[:b].astype(np.int64)
    ops.kv4_scatter(k, v, None, None, cuda(slots), kp, vp)
    assert ops.read_status() == 0
    ko.write(want[0], np64(k), slots, bs)
    ko.write(want[1], np64(v), slots, bs)
    assert np.array_equal(kp.cpu().numpy(), want[0]) and np.array_equal(vp.cpu().numpy(), want[1])


@pytest.mark.parametrize("layout", ["model", "heads_first", "offset"])
@pytest.mark.parametrize("b,h,d,bs,dtype", STORE)
def test_scatter_of_a_padded_source(b, h, d, bs, dtype, layout):
    """Tokens picked by row and position out of [B, H, L, D] views of three layouts; with "offset" the
    rows start one element past a 16-byte boundary."""
    rng = np.random.default_rng(d)
    length, n = 9, 11
    want = pools(rng, n, bs, h, d)
    kp, vp = cuda(want[0]), cuda(want[1])

    def source():
        x = tokens(rng, (b, length, h, d), dtype)
        if layout == "model":
            return x.transpose(1, 2)
        x = x.transpose(1, 2).contiguous()
        if layout == "heads_first":
            return x
        wide = torch.zeros((b, h, length, d + 1), dtype=x.dtype, device="cuda")
        wide[..., 1:] = x
        return wide[..., 1:]

    k, v = source(), source()
    rows = rng.integers(0, b, n).astype(np.int64)
    pos = rng.integers(0, length, n).astype(np.int64)
    slots = rng.permutation(n * bs)[:n].astype(np.int64)
    ops.kv4_scatter(k, v, cuda(rows), cuda(pos), cuda(slots), kp, vp)
    assert ops.read_status() == 0
    for pool, x in ((want[0], k), (want[1], v)):
        ko.write(pool, np64(x)[rows, :, pos], slots, bs)
    assert np.array_equal(kp.cpu().numpy(), want[0]) and np.array_equal(vp.cpu().numpy(), want[1])


@pytest.mark.parametrize("starts,lens,width", [([0, 5, 31], [16, 1, 7], 16), ([3], [1], 1), ([15, 16, 17, 0], [33, 32, 0, 40], 40)])
@pytest.mark.parametrize("h,d,bs,dtype", [(8, 128, 16, "bf16"), (2, 64, 3, "fp16"), (1, 32, 32, "bf16")])
def test_chunks_land_in_their_table_slots(starts, lens, width, h, d, bs, dtype):
    rng = np.random.default_rng(len(starts) + d)
    total = np.array(starts) + np.array(lens)
    tables, blocks = tables_for(rng, np.maximum(total, 1), bs)
    want = pools(rng, blocks, bs, h, d)
    kp, vp = cuda(want[0]), cuda(want[1])
    k = tokens(rng, (len(lens), width, h, d), dtype).transpose(1, 2)
    v = tokens(rng, (len(lens), width, h, d), dtype).transpose(1, 2)
    ops.kv4_store_chunks(k, v, torch.tensor(lens).cuda(), torch.tensor(starts).cuda(), cuda(tables), kp, vp)
    assert ops.read_status() == 0
    for pool, x in ((want[0], np64(k)), (want[1], np64(v))):
        for i, (st, n) in enumerate(zip(starts, lens)):
            slots = [tables[i, p // bs] * bs + p % bs for p in range(st, st + n)]
            if n:
                ko.write(pool, x[i, :, width - n :].transpose(1, 0, 2), slots, bs)
    assert np.array_equal(kp.cpu().numpy(), want[0]) and np.array_equal(vp.cpu().numpy(), want[1])


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_large_stores_meet_ties_and_near_ties(dtype):
    """A few million values on a coarse lattice with a sprinkling of tiny ones, which put quotients as near a
    tie as 16-bit sources can without meeting it: every code is the oracle's."""
    rng = np.random.default_rng(11)
    b, h, d, bs = 2000, 8, 128, 16
    x = rng.standard_normal((b, h, d)) * 1.3
    x = np.where(rng.random(x.shape) < 0.02, x * 10.0 ** rng.uniform(-6, -3, x.shape), x)
    k = torch.from_numpy(x).to(DTYPES[dtype]).cuda()
    kp = torch.zeros((b // bs, h, ops.kv4_page_bytes(bs, d)), dtype=torch.uint8, device="cuda")
    vp = torch.zeros_like(kp)
    ops.kv4_scatter(k, k.flip(0), None, None, torch.arange(b).cuda(), kp, vp)
    want = ko.stored(np64(k))
    got = ko.read(kp.cpu().numpy(), range(b // bs), bs, d).reshape(b, h, d)
    other = ko.read(vp.cpu().numpy(), range(b // bs), bs, d).reshape(b, h, d)
    # x - m and its quotient (at most 15.1) are each rounded by 2^-24 at most: only a quotient nearer a tie than
    # 15.1 * 2^-23, and not on it, may go the other way
    _, s, m = ko.quantise(np64(k))
    exact = (np64(k).reshape(b, h, -1, ko.GROUP) - m[..., None]) / s[..., None].astype(np.float64)
    away = np.abs(exact - np.floor(exact) - 0.5).reshape(x.shape)
    assert not ((got != want) & ((away == 0) | (away > 15.1 * 2.0**-23))).any()
    assert np.array_equal(other[::-1], got)


def test_store_of_32_bit_sources_is_at_most_a_near_tie_away():
    """fp32 sources: x - m and its quotient are rounded, so a code may differ where the exact quotient is
    within 15 * 2^-22 of a tie (two roundings of at most 2^-24 relative, on a quotient up to 15)."""
    rng = np.random.default_rng(1)
    b, h, d, bs = 64, 4, 128, 16
    k = torch.from_numpy(rng.standard_normal((b, h, d)).astype(np.float32)).cuda()
    kp = torch.zeros((5, h, ops.kv4_page_bytes(bs, d)), dtype=torch.uint8, device="cuda")
    vp = torch.zeros_like(kp)
    ops.kv4_scatter(k, k, None, None, torch.arange(b).cuda(), kp, vp)
    c, s, m = ko.quantise(np64(k))
    got = ko.read(kp.cpu().numpy(), range(4), bs, d).reshape(b, h, -1, ko.GROUP)
    exact = (np64(k).reshape(got.shape) - m[..., None]) / s[..., None]
    off = np.rint((got - m[..., None]) / s[..., None]) - c
    tie = np.abs(exact - np.floor(exact) - 0.5) < 15 * 2.0**-22
    assert (off[~tie] == 0).all() and np.abs(off).max() <= 1
    assert torch.equal(kp, vp)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_values_no_group_describes_read_back_as_nan(dtype):
    """An infinity or a NaN takes its group of 32 with it and no other; a constant group is kept to bfloat16."""
    h, d, bs = 2, 64, 16
    k = torch.zeros((4, h, d), dtype=DTYPES[dtype], device="cuda")
    k[0, 0, 3], k[1, 1, 40], k[2, 0, 0] = float("inf"), float("nan"), float("-inf")
    k[3, 1] = -2.5
    kp = torch.zeros((1, h, ops.kv4_page_bytes(bs, d)), dtype=torch.uint8, device="cuda")
    vp = torch.zeros_like(kp)
    ops.kv4_scatter(k, k, None, None, torch.arange(4).cuda(), kp, vp)
    got, _ = ops.kv4_gather_blocks(kp, vp, torch.zeros((1, 1), dtype=torch.long).cuda(), d, DTYPES[dtype])
    got = got[0, 0]
    want = torch.zeros((bs, h, d), dtype=DTYPES[dtype], device="cuda")
    want[0, 0, :32] = want[1, 1, 32:] = want[2, 0, :32] = float("nan")
    want[3, 1] = -2.5
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got.nan_to_num(), want.nan_to_num())


def test_a_store_touches_nothing_else():
    rng = np.random.default_rng(0)
    h, d, bs = 3, 128, 16
    kp = torch.full((4, h, ops.kv4_page_bytes(bs, d)), 0xA5, dtype=torch.uint8, device="cuda")
    vp = kp.clone()
    k = tokens(rng, (1, h, d), "bf16")
    ops.kv4_scatter(k, k, None, None, torch.tensor([37]).cuda(), kp, vp)  # block 2, offset 5
    ng = d // 32
    touched = torch.zeros_like(kp, dtype=torch.bool)
    for g in range(ng):
        touched[2, :, (g * bs + 5) * 16 : (g * bs + 6) * 16] = True
    touched[2, :, ng * bs * 16 + 5 * ng * 4 : ng * bs * 16 + 6 * ng * 4] = True
    assert (kp[~touched] == 0xA5).all() and (vp[~touched] == 0xA5).all()


def test_bad_slots_rows_lengths_and_blocks_are_flagged_and_skipped():
    rng = np.random.default_rng(2)
    h, d, bs, n = 2, 64, 4, 3
    k = tokens(rng, (4, h, d), "bf16")
    kp = torch.zeros((n, h, ops.kv4_page_bytes(bs, d)), dtype=torch.uint8, device="cuda")
    vp = torch.zeros_like(kp)
    ops.kv4_scatter(k, k, None, None, torch.tensor([-1, n * bs, 1 << 40, -(1 << 40)]).cuda(), kp, vp)
    assert ops.read_status() == nat.MI_STATUS_BAD_SLOT and not kp.any() and not vp.any()
    x = k[:, :, None]
    ops.kv4_scatter(x, x, torch.tensor([4, 0]).cuda(), torch.tensor([0, 1]).cuda(), torch.tensor([0, 1]).cuda(), kp, vp)
    assert ops.read_status() == nat.MI_STATUS_BAD_INDEX and not kp.any()
    one = torch.ones(4, dtype=torch.long).cuda()
    tables = torch.tensor([[1], [n], [-1], [2]]).cuda()
    ops.kv4_store_chunks(x, x, one, torch.tensor([0, 0, 0, 4]).cuda(), tables, kp, vp)
    assert ops.read_status() == nat.MI_STATUS_BAD_BLOCK | nat.MI_STATUS_BAD_LENGTH
    assert kp[1].any() and not kp[0].any() and not kp[2].any()
    key, value = ops.kv4_gather_blocks(kp, vp, torch.tensor([[1, n], [-7, 0]]).cuda(), d, torch.bfloat16)
    assert ops.read_status() == nat.MI_STATUS_BAD_BLOCK
    assert key[0, 0].any() and not key[0, 1].any() and not key[1].any() and not value[1].any()


@pytest.mark.parametrize("d", [32, 64, 128, 256])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_append_fused_with_norm_and_rope_leaves_the_scatters_bytes(d, dtype):
    """Against mi_qk_norm_rope's own outputs scattered, q included; packed projections, a bad slot, a NaN."""
    rng = np.random.default_rng(d)
    t, hq, h, bs, n = 7, 4, 2, 16, 3
    qkv = tokens(rng, (t, (hq + 2 * h) * d), dtype)
    q, k, v = qkv[:, : hq * d], qkv[:, hq * d : (hq + h) * d], qkv[:, (hq + h) * d :]
    v[3, 5] = float("nan")
    v[4] = 0.5
    qw, kw = tokens(rng, (d,), dtype), tokens(rng, (d,), dtype)
    cos, sin = tokens(rng, (t, d), dtype), tokens(rng, (t, d), dtype)
    slots = torch.tensor([5, 17, 0, 47, 30, 31, n * bs]).cuda()
    fused = [torch.zeros((n, h, ops.kv4_page_bytes(bs, d)), dtype=torch.uint8, device="cuda") for _ in range(2)]
    apart = [p.clone() for p in fused]
    got = ops.kv4_qk_norm_rope(q, k, v, qw, kw, cos, sin, 1e-6, hq, h, slots, *fused)
    assert ops.read_status() == nat.MI_STATUS_BAD_SLOT
    want, k_out, v_out = ops.qk_norm_rope(q, k, v, qw, kw, cos, sin, 1e-6, hq, h)
    ops.kv4_scatter(k_out[:6], v_out[:6], None, None, slots[:6], *apart)
    assert ops.read_status() == 0
    assert torch.equal(got, want) and torch.equal(fused[0], apart[0]) and torch.equal(fused[1], apart[1])
    for args in [(q, k, v, qw, kw, cos, sin, 1e-6, hq, h, slots[:6], *fused),
                 (q, k[:, :d], v, qw, kw, cos, sin, 1e-6, hq, h, slots, *fused),
                 (q, k, v, qw, kw, cos[:3], sin[:3], 1e-6, hq, h, slots, *fused),
                 (q, k, v, qw, kw, cos.double(), sin, 1e-6, hq, h, slots, *fused),
                 (q, k, v, qw, kw, cos, sin, 1e-6, hq, h, slots, fused[0][:, :1], fused[1][:, :1])]:
        with pytest.raises(ValueError):
            ops.kv4_qk_norm_rope(*args)


# ---------------------------------------------------------------------------------------------
# gather
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("h,d,bs,dtype", [(8, 128, 16, "bf16"), (2, 64, 16, "fp16"), (1, 32, 3, "fp32"), (3, 96, 1, "bf16"),
                                          (2, 256, 32, "fp16")])
@pytest.mark.parametrize("lengths", [None, [0, 1, 48, 17], [48, 47, 33, 16]])
def test_gather_is_the_values_rounded_once(h, d, bs, dtype, lengths):
    """m + s * c rounded once to bf16 or fp32; to fp16 twice (fp32 first), so it may be off by half a unit
    and 2^-24 of the value."""
    rng = np.random.default_rng(d + bs)
    nb, b, blocks = 48 // bs + 1, 4, 9
    kp, vp = pools(rng, blocks, bs, h, d)
    ids = rng.integers(0, blocks, (b, nb)).astype(np.int64)
    lens = None
    if lengths is not None:
        lens = torch.tensor(lengths).cuda()
        for i, n in enumerate(lengths):  # ids past a row's length are never read
            ids[i, -(-n // bs) :] = blocks + 5
        kp_n, vp_n = kp.copy(), vp.copy()
    gk, gv = ops.kv4_gather_blocks(cuda(kp), cuda(vp), cuda(ids), d, DTYPES[dtype], lengths=lens)
    assert ops.read_status() == 0 and gk.shape == (b, nb, bs, h, d)
    for got, pool in ((gk, kp), (gv, vp)):
        want = ko.read(pool, np.minimum(ids, blocks - 1).reshape(-1), bs, d).reshape(b, nb * bs, h, d)
        if lengths is not None:
            for i, n in enumerate(lengths):
                want[i, n:] = 0
        g = np64(got).reshape(b, nb * bs, h, d)
        ulp = torch.finfo(DTYPES[dtype]).eps * np.abs(want)
        assert (np.abs(g - want) <= 0.5 * ulp * (1 + 2.0**-9) + 1e-30).all()
        assert ((want == 0) <= (g == 0)).all()


def test_gather_zeros_what_a_page_holds_past_the_length():
    """Stale NaN parameters past a row's length do not come back."""
    d, bs, h = 128, 16, 2
    kp = torch.full((3, h, ops.kv4_page_bytes(bs, d)), 0xFF, dtype=torch.uint8, device="cuda")
    rng = np.random.default_rng(3)
    k = tokens(rng, (5, h, d), "bf16")
    vp = kp.clone()
    ops.kv4_scatter(k, k, None, None, torch.arange(16, 21).cuda(), kp, vp)
    key, value = ops.kv4_gather_blocks(kp, vp, torch.tensor([[1, 2]]).cuda(), d, torch.bfloat16,
                                       lengths=torch.tensor([5]).cuda())
    assert torch.isfinite(key).all() and torch.isfinite(value).all()
    assert key[0, 0, :5].any() and not key[0, 0, 5:].any() and not key[0, 1].any()


def test_ids_that_are_a_column_slice():
    rng = np.random.default_rng(4)
    kp, vp = (cuda(p) for p in pools(rng, 6, 16, 2, 64))
    ids = torch.tensor([[1, 2, 3, 4], [5, 4, 3, 2]]).cuda()
    part, _ = ops.kv4_gather_blocks(kp, vp, ids[:, 1:3], 64, torch.float16)
    whole, _ = ops.kv4_gather_blocks(kp, vp, ids, 64, torch.float16)
    assert torch.equal(part, whole[:, 1:3])


# ---------------------------------------------------------------------------------------------
# decode
# ---------------------------------------------------------------------------------------------
def decode_tolerance(want, q, kp, vp, tables, ctx, scale, bs, dtype):
    """A bound on |decode - exact| per row, from the roundings the operator may make:

    * the output's: half a unit, eps/2 * |o| (2^-25 below fp16's normal range);
    * p * s in fp16 (16-bit types): at most half a unit, 2^-11, of p * s * c, and s * c <= R = the widest
      15 * s of the row's values; fp16 models carry the remainder in a second fp16: 2^-22;
    * fp32 sums: a score is a sum of 2 * D terms within 2^-24 each (its operands are exact or, far below
      the row's largest, within 2^-24 of it), so it is off by at most d = (2 D + 64) 2^-24 scale sum|q||k|,
      a weight by a factor e^d and 2^-21 for the exponential, and the output by twice that times max|v|;
      the two sums over the tokens by (n + 64) 2^-24 max|v| each.
    """
    b, hq, d = q.shape
    h = kp.shape[1]
    tol = np.zeros((b, hq, 1))
    unit = {"bf16": 2.0**-11, "fp16": 2.0**-22, "fp32": 0.0}[dtype]
    for i in range(b):
        n = int(ctx[i])
        if n <= 0:
            continue
        ids = tables[i, : -(-n // bs)]
        k = np.abs(ko.read(kp, ids, bs, d).reshape(-1, h, d)[:n]).repeat(hq // h, axis=1)
        v = ko.read(vp, ids, bs, d).reshape(-1, h, d)[:n]
        big = np.abs(v).max(axis=(0, 2)).repeat(hq // h)[:, None]
        group = v.reshape(n, h, -1, ko.GROUP)
        wide = (group.max(-1) - group.min(-1)).max(axis=(0, 2)).repeat(hq // h)[:, None]
        delta = (2 * d + 64) * 2.0**-24 * scale * np.einsum("hd,thd->ht", np.abs(q[i]), k).max(-1, keepdims=True)
        tol[i] = unit * wide * 1.07 + (2 * (np.expm1(delta) + 2.0**-21) + 2 * (n + 64) * 2.0**-24) * big
    half = torch.finfo(DTYPES[dtype]).eps / 2
    return tol.repeat(d, axis=2).reshape(b, hq * d) + half * np.abs(want) * 1.01 + (2.0**-25 if dtype == "fp16" else 1e-30)


DECODE = [
    # batch, query heads, KV heads, head_dim, block size, lengths (lo, hi), dtype
    (5, 16, 8, 128, 16, (1, 300), "bf16"),    # two query heads a KV head, four KV heads a CTA
    (3, 32, 8, 128, 16, (200, 1500), "bf16"),  # four
    (4, 8, 1, 128, 16, (1, 2100), "bf16"),    # eight, one KV head
    (3, 8, 2, 128, 32, (30, 900), "fp16"),    # two KV heads, wider blocks
    (7, 12, 6, 64, 16, (1, 333), "fp16"),
    (3, 5, 5, 128, 16, (100, 257), "bf16"),   # one query head a KV head, an odd number of them
    (2, 6, 2, 64, 32, (33, 70), "bf16"),      # three a KV head
    (9, 14, 2, 128, 16, (1, 40), "fp16"),     # seven
    (2, 32, 2, 128, 16, (50, 300), "bf16"),   # sixteen: past the tensor tile
    (4, 4, 2, 32, 3, (1, 50), "fp32"),
    (3, 4, 4, 96, 1, (1, 20), "bf16"),
    (2, 4, 1, 256, 16, (40, 70), "fp16"),
    (3, 6, 3, 160, 4, (1, 30), "fp32"),
    (2, 8, 4, 128, 48, (1, 200), "bf16"),
]


def decode_case(b, hq, h, d, bs, lengths, dtype, seed=0):
    rng = np.random.default_rng(seed + b + hq + d + bs)
    ctx = rng.integers(lengths[0], lengths[1] + 1, b).astype(np.int64)
    ctx[0] = lengths[1]
    tables, blocks = tables_for(rng, ctx, bs)
    kp, vp = pools(rng, blocks, bs, h, d)
    q = tokens(rng, (b, hq, d), dtype)
    return q, kp, vp, tables, ctx


@pytest.mark.parametrize("b,hq,h,d,bs,lengths,dtype", DECODE)
def test_decode_matches_the_oracle(b, hq, h, d, bs, lengths, dtype):
    q, kp, vp, tables, ctx = decode_case(b, hq, h, d, bs, lengths, dtype)
    scale = d**-0.5
    got = ops.kv4_paged_decode(q, cuda(kp), cuda(vp), cuda(tables), cuda(ctx), scale)
    assert ops.read_status() == 0 and got.shape == (b, hq * d) and got.dtype == q.dtype
    want = ko.decode(np64(q), kp, vp, tables, ctx, scale, bs)
    err = np.abs(np64(got) - want)
    tol = decode_tolerance(want, np64(q), kp, vp, tables, ctx, scale, bs, dtype)
    assert (err <= tol).all(), f"{(err / tol).max():.2f} of the tolerance"


CUT = [
    # batch, query heads, KV heads, head_dim, block size, longest, dtype: sequences cut over many CTAs, CTAs
    # that hold many sequences, rows of no tokens between them
    (1, 8, 1, 128, 16, 9000, "bf16"),
    (1, 4, 2, 64, 32, 20011, "fp16"),
    (2, 4, 4, 128, 16, 7001, "bf16"),
    (300, 4, 1, 64, 16, 700, "bf16"),
    (40, 8, 4, 128, 16, 1700, "fp16"),
    (700, 2, 2, 64, 16, 90, "bf16"),     # short tables: whole sequences
    (1000, 1, 1, 64, 16, 400, "bf16"),
]


@pytest.mark.parametrize("b,hq,h,d,bs,longest,dtype", CUT)
def test_decode_of_streams_that_are_cut(b, hq, h, d, bs, longest, dtype):
    rng = np.random.default_rng(b + longest)
    ctx = np.minimum(rng.geometric(4 / longest, b), longest).astype(np.int64)
    ctx[rng.integers(b)] = longest
    if b > 2:
        ctx[rng.integers(0, b, b // 8)] = 0
        ctx[[0, -1]] = 0
    # pages shared by all rows: what counts here is who takes which steps
    blocks = 64
    kp, vp = pools(rng, blocks, bs, h, d)
    tables = rng.integers(1, blocks, (b, -(-longest // bs))).astype(np.int64)
    q = tokens(rng, (b, hq, d), dtype)
    scale = d**-0.5
    got = ops.kv4_paged_decode(q, cuda(kp), cuda(vp), cuda(tables), cuda(ctx), scale)
    assert ops.read_status() == 0
    want = ko.decode(np64(q), kp, vp, tables, ctx, scale, bs)
    tol = decode_tolerance(want, np64(q), kp, vp, tables, ctx, scale, bs, dtype)
    err = np.abs(np64(got) - want)
    assert (err <= tol).all(), f"{(err / tol).max():.2f} of the tolerance"
    assert not got[torch.from_numpy(ctx == 0).cuda()].any()
    again = ops.kv4_paged_decode(q, cuda(kp), cuda(vp), cuda(tables), cuda(ctx), scale)
    assert torch.equal(got, again)


@pytest.mark.parametrize("width", [3, 60])
def test_bad_blocks_and_lengths_whole_or_cut(width):
    """Flags and clamps on tables short enough for whole sequences and on longer ones, whose stream is cut."""
    rng = np.random.default_rng(width)
    b, hq, h, d, bs, blocks = 6, 8, 4, 128, 16, 20
    kp, vp = (cuda(p) for p in pools(rng, blocks, bs, h, d))
    q = tokens(rng, (b, hq, d), "bf16")
    tables = rng.integers(1, blocks, (b, width)).astype(np.int64)
    ctx = np.full(b, width * bs - 5, dtype=np.int64)
    fine = ops.kv4_paged_decode(q, kp, vp, cuda(tables), cuda(ctx), 0.1)
    bad, null = tables.copy(), tables.copy()
    bad[1, 0], bad[3, width - 1], bad[4, 1] = -1, blocks, 1 << 60
    null[1, 0] = null[3, width - 1] = null[4, 1] = 0
    out = ops.kv4_paged_decode(q, kp, vp, cuda(bad), cuda(ctx), 0.1)
    assert ops.read_status() == nat.MI_STATUS_BAD_BLOCK
    assert torch.equal(out, ops.kv4_paged_decode(q, kp, vp, cuda(null), cuda(ctx), 0.1))
    assert torch.equal(out[[0, 2, 5]], fine[[0, 2, 5]])
    over = ctx.copy()
    over[2], over[5] = width * bs + 1, 1 << 62
    out = ops.kv4_paged_decode(q, kp, vp, cuda(tables), cuda(over), 0.1)
    assert ops.read_status() == nat.MI_STATUS_BAD_LENGTH
    over[[2, 5]] = width * bs
    assert torch.equal(out, ops.kv4_paged_decode(q, kp, vp, cuda(tables), cuda(over), 0.1))
    over[[0, 3]] = -(1 << 62)
    out = ops.kv4_paged_decode(q, kp, vp, cuda(tables), cuda(over), 0.1)
    assert not out[[0, 3]].any() and ops.read_status() == 0


@pytest.mark.parametrize("d,bs,dtype", [(128, 16, "bf16"), (64, 32, "fp16"), (128, 32, "bf16"), (32, 5, "fp32")])
def test_decode_at_every_length_of_a_page_and_none(d, bs, dtype):
    """Lengths 0 to two pages and one token in one batch, pages poisoned past every length: a row of none
    gives zeros, no row sees what lies past its end."""
    rng = np.random.default_rng(d)
    h, g = 2, 2
    ctx = np.arange(2 * bs + 2).astype(np.int64)
    tables, blocks = tables_for(rng, np.maximum(ctx, 1), bs)
    kp, vp = (np.full((blocks, h, ko.page_bytes(bs, d)), 0xFF, dtype=np.uint8) for _ in range(2))
    for i, n in enumerate(ctx):
        slots = [tables[i, p // bs] * bs + p % bs for p in range(n)]
        for pool in (kp, vp):
            if n:
                ko.write(pool, np64(tokens(rng, (int(n), h, d), "bf16")), slots, bs)
    q = tokens(rng, (len(ctx), h * g, d), dtype)
    got = ops.kv4_paged_decode(q, cuda(kp), cuda(vp), cuda(tables), cuda(ctx), 0.3)
    assert ops.read_status() == 0
    want = ko.decode(np64(q), kp, vp, tables, ctx, 0.3, bs)
    tol = decode_tolerance(want, np64(q), kp, vp, tables, ctx, 0.3, bs, dtype)
    assert (np.abs(np64(got) - want) <= tol).all()
    assert not got[0].any()


@pytest.mark.parametrize("scale_k,scale_v,dtype", [(40.0, 1.0, "bf16"), (1e-4, 1e-9, "bf16"), (3.0, 3e4, "bf16"),
                                                   (1.0, 1e-3, "fp16"), (30.0, 100.0, "fp16")])
def test_decode_over_wide_ranges_of_keys_and_values(scale_k, scale_v, dtype):
    """Peaked and flat softmaxes, value steps far from one, growing along the sequence so that every
    running reference has to move, and one token with constant (step 0) values that takes most weight."""
    rng = np.random.default_rng(int(scale_k))
    b, hq, h, d, bs, n = 2, 8, 2, 128, 16, 700
    ctx = np.array([n, n - 37], dtype=np.int64)
    tables, blocks = tables_for(rng, ctx, bs)
    kp, vp = (np.zeros((blocks, h, ko.page_bytes(bs, d)), dtype=np.uint8) for _ in range(2))
    for i in range(b):
        m = int(ctx[i])
        slots = [tables[i, p // bs] * bs + p % bs for p in range(m)]
        ramp = np.geomspace(1e-2, 1, m)[:, None, None]
        ko.write(kp, rng.standard_normal((m, h, d)) * scale_k * ramp, slots, bs)
        v = rng.standard_normal((m, h, d)) * scale_v * ramp
        v[m // 2] = scale_v
        ko.write(vp, v, slots, bs)
    q = tokens(rng, (b, hq, d), dtype)
    got = ops.kv4_paged_decode(q, cuda(kp), cuda(vp), cuda(tables), cuda(ctx), d**-0.5)
    want = ko.decode(np64(q), kp, vp, tables, ctx, d**-0.5, bs)
    tol = decode_tolerance(want, np64(q), kp, vp, tables, ctx, d**-0.5, bs, dtype)
    assert (np.abs(np64(got) - want) <= tol).all()


def test_decode_with_the_append_is_the_append_then_the_decode():
    q, kp, vp, tables, ctx = decode_case(6, 16, 8, 128, 16, (1, 400), "bf16")
    rng = np.random.default_rng(7)
    kn, vn = tokens(rng, (6, 8, 128), "bf16"), tokens(rng, (6, 8, 128), "bf16")
    slots = np.array([tables[i, (c - 1) // 16] * 16 + (c - 1) % 16 for i, c in enumerate(ctx)], dtype=np.int64)
    a, b, c, d = cuda(kp), cuda(vp), cuda(kp), cuda(vp)
    one = ops.kv4_paged_decode(q, a, b, cuda(tables), cuda(ctx), 0.1, key_new=kn, value_new=vn, slot_mapping=cuda(slots))
    ops.kv4_scatter(kn, vn, None, None, cuda(slots), c, d)
    two = ops.kv4_paged_decode(q, c, d, cuda(tables), cuda(ctx), 0.1)
    assert torch.equal(one, two) and torch.equal(a, c) and torch.equal(b, d) and not torch.equal(a, cuda(kp))
    ko.write(kp, np64(kn), slots, 16)
    assert np.array_equal(a.cpu().numpy(), kp)


@pytest.mark.parametrize("d,dtype", [(128, "bf16"), (64, "fp16")])
def test_decode_of_strided_operands(d, dtype):
    """Query rows of a packed projection, tables that are a column slice, an output inside wider rows."""
    q, kp, vp, tables, ctx = decode_case(5, 8, 4, d, 16, (1, 200), dtype)
    kp, vp, ctx = cuda(kp), cuda(vp), cuda(ctx)
    want = ops.kv4_paged_decode(q, kp, vp, cuda(tables), ctx, 0.2)
    packed = torch.zeros((5, 8 * d + 96 + 2), dtype=q.dtype, device="cuda")
    packed[:, 2 : 2 + 8 * d] = q.view(5, -1)
    wide = torch.zeros((5, tables.shape[1] + 3), dtype=torch.long, device="cuda")
    wide[:, : tables.shape[1]] = cuda(tables)
    out = torch.full((5, 8 * d + 6), 7.0, dtype=q.dtype, device="cuda")
    got = ops.kv4_paged_decode(packed[:, 2 : 2 + 8 * d].view(5, 8, d), kp, vp, wide[:, : tables.shape[1]], ctx, 0.2,
                               out=out[:, 3 : 3 + 8 * d])
    assert torch.equal(got, want)
    assert (out[:, :3] == 7).all() and (out[:, 3 + 8 * d :] == 7).all()


def test_decode_flags_bad_blocks_and_lengths_and_stays_in_bounds():
    q, kp, vp, tables, ctx = decode_case(3, 8, 4, 128, 16, (40, 60), "bf16")
    kp, vp = cuda(kp), cuda(vp)
    bad = tables.copy()
    bad[0, 1], bad[1, 0] = kp.shape[0], -3
    out = ops.kv4_paged_decode(q, kp, vp, cuda(bad), cuda(ctx), 0.1)
    assert ops.read_status() == nat.MI_STATUS_BAD_BLOCK and torch.isfinite(out).all()
    null = tables.copy()
    null[0, 1] = null[1, 0] = 0
    assert torch.equal(out, ops.kv4_paged_decode(q, kp, vp, cuda(null), cuda(ctx), 0.1))
    long = ctx.copy()
    long[2] = 10**12
    ops.kv4_paged_decode(q, kp, vp, cuda(tables), cuda(long), 0.1)
    assert ops.read_status() == nat.MI_STATUS_BAD_LENGTH
    minus = ctx.copy()
    minus[1] = -5
    assert not ops.kv4_paged_decode(q, kp, vp, cuda(tables), cuda(minus), 0.1)[1].any()
    assert ops.read_status() == 0


def test_decode_repeats_bit_for_bit():
    q, kp, vp, tables, ctx = decode_case(6, 16, 8, 128, 16, (500, 3000), "bf16")
    args = cuda(kp), cuda(vp), cuda(tables), cuda(ctx)
    first = ops.kv4_paged_decode(q, *args, 0.09)
    for _ in range(3):
        assert torch.equal(first, ops.kv4_paged_decode(q, *args, 0.09))


def test_nan_of_one_sequence_stays_there():
    q, kp, vp, tables, ctx = decode_case(3, 8, 4, 128, 16, (20, 40), "bf16")
    kp, vp = cuda(kp), cuda(vp)
    clean = ops.kv4_paged_decode(q, kp, vp, cuda(tables), cuda(ctx), 0.1)
    k = torch.zeros((1, 4, 128), dtype=torch.bfloat16, device="cuda")
    k[0, 1, 5] = float("nan")
    ops.kv4_scatter(k, k, None, None, torch.tensor([int(tables[1, 0]) * 16 + 2]).cuda(), kp, vp)
    got = ops.kv4_paged_decode(q, kp, vp, cuda(tables), cuda(ctx), 0.1).view(3, 4, 2, 128)
    assert torch.equal(got[[0, 2]], clean.view(3, 4, 2, 128)[[0, 2]])
    assert torch.isnan(got[1, 1]).all() and torch.isfinite(got[1, [0, 2, 3]]).all()


def test_two_streams_and_a_captured_graph_share_no_workspace():
    """Two decodes at once on two streams, and a graph replayed while an eager call runs."""
    a = decode_case(2, 8, 1, 128, 16, (3000, 4000), "bf16", seed=1)
    b = decode_case(2, 8, 1, 128, 16, (3000, 4000), "bf16", seed=2)
    args = [(x[0], cuda(x[1]), cuda(x[2]), cuda(x[3]), cuda(x[4]), 0.1) for x in (a, b)]
    want = [ops.kv4_paged_decode(*x) for x in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        got = []
        for s, x in zip(streams, args):
            with torch.cuda.stream(s):
                got.append(ops.kv4_paged_decode(*x))
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graphs, outs = [], []
    for x in args:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.kv4_paged_decode(*x))
        graphs.append(g)
    for _ in range(5):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        again = ops.kv4_paged_decode(*args[0])
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]) and torch.equal(again, want[0])


def test_the_ordinary_call_and_the_general_one_agree():
    """Plain contiguous operands go through the CPython extension, others (here: an output of one's own, a
    strided id or length tensor, index tensors) through ctypes: the same results, bit for bit."""
    q, kp, vp, tables, ctx = decode_case(6, 16, 8, 128, 16, (1, 900), "bf16")
    kp, vp, tables, ctx = cuda(kp), cuda(vp), cuda(tables), cuda(ctx)
    calls = nat.calls()
    quick = calls.kv4_paged_decode(q, kp, vp, tables, ctx, 0.1)
    assert quick is not None
    assert torch.equal(quick, ops.kv4_paged_decode(q, kp, vp, tables, ctx, 0.1, out=torch.empty_like(quick)))
    ids = tables[:, :3].contiguous()
    wide = torch.zeros((6, 6), dtype=torch.long, device="cuda")
    wide[:, ::2] = ids
    quick = calls.kv4_gather_blocks(kp, vp, ids, 128, nat.MI_F16, ctx, True)
    assert calls.kv4_gather_blocks(kp, vp, wide[:, ::2], 128, nat.MI_F16, ctx, True) is None
    general = ops.kv4_gather_blocks(kp, vp, wide[:, ::2], 128, torch.float16, lengths=ctx)
    assert torch.equal(quick[0], general[0]) and torch.equal(quick[1], general[1])
    k = q[:, :8]
    slots, rows = torch.arange(6).cuda(), torch.arange(6).cuda()
    a, b = [kp.clone(), vp.clone()], [kp.clone(), vp.clone()]
    assert calls.kv4_append(k, k, slots, *a)
    ops.kv4_scatter(k[:, :, None], k[:, :, None], rows, None, slots, *b)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    x = k[:, :, None]
    one = torch.ones(6, dtype=torch.long, device="cuda")
    spread = torch.ones(12, dtype=torch.long, device="cuda")[::2]
    own = torch.arange(1, 7).cuda()[:, None]
    assert calls.kv4_store_chunks(x, x, one, one, own, *a)
    assert calls.kv4_store_chunks(x, x, spread, one, own, *b) is None
    ops.kv4_store_chunks(x, x, spread, one, own, *b)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    pairs = torch.tensor([[1, 8], [2, 9]]).cuda()
    assert calls.kv_copy_blocks(a, pairs) and calls.kv_copy_blocks(iter(b), pairs) is None
    ops.kv_copy_blocks(b, pairs.t().contiguous().t())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    for bad in [(q.cpu(), kp, vp, tables, ctx, 0.1), (q, kp, vp, tables.int(), ctx, 0.1), (q, kp, vp, tables, ctx[:3], 0.1),
                (q, kp, kp[:1], tables, ctx, 0.1), (q, kp, vp, tables, ctx, "x"), (None, kp, vp, tables, ctx, 0.1), (q,)]:
        assert calls.kv4_paged_decode(*bad) is None
    assert calls.kv4_gather_blocks(kp, vp, ids, "d", nat.MI_F16, ctx, True) is None
    assert ops.read_status() == 0


def test_weights_outputs_and_workspaces_of_another_form_are_refused():
    """Each would be read or written as if it were contiguous [D], distinct rows or a plain run of bytes."""
    d, hq, h, bs, n = 64, 4, 2, 16, 3
    x = torch.zeros((2, hq * d), dtype=torch.bfloat16, device="cuda")
    w = torch.ones(2 * d, dtype=torch.bfloat16, device="cuda")
    cos, slots = x[:, :d], torch.tensor([0, 1]).cuda()
    pools = [torch.zeros((n, h, ops.kv4_page_bytes(bs, d)), dtype=torch.uint8, device="cuda") for _ in range(2)]
    for qw, kw in [(w[:d], w[: d // 2]), (w[:d], w[::2]), (w[::2], w[:d]), (w[:d], w[:d, None])]:
        with pytest.raises(ValueError, match="weight"):
            ops.kv4_qk_norm_rope(x, x[:, : h * d], x[:, : h * d], qw, kw, cos, cos, 1e-6, hq, h, slots, *pools)
    q, ctx = x.view(2, hq, d), torch.ones(2, dtype=torch.long, device="cuda")
    tables = torch.ones((2, 40), dtype=torch.long, device="cuda")
    with pytest.raises(ValueError, match="out"):
        ops.kv4_paged_decode(q, *pools, tables, ctx, 1.0, out=x[:1].expand(2, hq * d))
    with pytest.raises(ValueError, match="ws"):
        ops.kv4_paged_decode(q, *pools, tables, ctx, 1.0, ws=torch.zeros(1 << 25, dtype=torch.uint8, device="cuda")[::2])


# ---------------------------------------------------------------------------------------------
# refusals
# ---------------------------------------------------------------------------------------------
def test_refusals():
    d, bs, h, n = 64, 16, 2, 4
    page = ops.kv4_page_bytes(bs, d)
    kp = torch.zeros((n, h, page), dtype=torch.uint8, device="cuda")
    vp = torch.zeros_like(kp)
    k = torch.zeros((2, h, d), dtype=torch.bfloat16, device="cuda")
    slots = torch.tensor([0, 1]).cuda()
    tables, ctx = torch.zeros((2, 3), dtype=torch.long).cuda(), torch.ones(2, dtype=torch.long).cuda()
    q = torch.zeros((2, 4, d), dtype=torch.bfloat16, device="cuda")
    for args in [
        (k[..., :48], k[..., :48], None, None, slots, kp, vp),  # head_dim not a multiple of 32
        (k, k[:, :, :32], None, None, slots, kp, vp),
        (k, k.half(), None, None, slots, kp, vp),
        (k[:, :1], k[:, :1], None, None, slots, kp, vp),
        (k, k, None, None, slots.int(), kp, vp),
        (k, k, None, None, torch.arange(3).cuda(), kp, vp),
        (k, k, slots, None, slots, kp, vp),
        (k, k, None, None, slots, kp.view(torch.int8), vp),
        (k, k, None, None, slots, kp[:, :, : page - 1], vp),
        (k, k, None, None, slots, torch.zeros((n, h, page + 1), dtype=torch.uint8).cuda(),
         torch.zeros((n, h, page + 1), dtype=torch.uint8).cuda()),
        (k.double(), k.double(), None, None, slots, kp, vp),
    ]:
        with pytest.raises(ValueError):
            ops.kv4_scatter(*args)
    x = k[:, :, None]
    for args in [(k, k, ctx, ctx, tables, kp, vp), (x, x, ctx[:1], ctx, tables, kp, vp),
                 (x, x, ctx, ctx, tables[:1], kp, vp), (x, x, ctx, ctx, tables.int(), kp, vp),
                 (x[:, :1], x[:, :1], ctx, ctx, tables, kp, vp)]:
        with pytest.raises(ValueError):
            ops.kv4_store_chunks(*args)
    for args, more in [((kp, vp, tables, 96, torch.bfloat16), {}), ((kp, vp, tables, d, torch.float64), {}),
                       ((kp, vp, tables.int(), d, torch.bfloat16), {}), ((kp, vp, ctx, d, torch.bfloat16), {}),
                       ((kp, vp, tables, d, torch.bfloat16), {"lengths": ctx[:1]})]:
        with pytest.raises(ValueError):
            ops.kv4_gather_blocks(*args, **more)
    for args, more in [
        ((q[0], kp, vp, tables, ctx, 1.0), {}),
        ((q[:, :3], kp, vp, tables, ctx, 1.0), {}),
        ((q, kp, vp, tables[:1], ctx, 1.0), {}),
        ((q, kp, vp, tables[:, :0], ctx, 1.0), {}),
        ((q, kp, vp, tables, ctx[:1], 1.0), {}),
        ((q, kp, vp, tables, ctx, 1.0), {"key_new": k}),
        ((q, kp, vp, tables, ctx, 1.0), {"key_new": k.half(), "value_new": k.half(), "slot_mapping": slots}),
        ((q, kp, vp, tables, ctx, 1.0), {"out": torch.zeros((2, 4 * d), device="cuda")}),
        ((q.double(), kp, vp, tables, ctx, 1.0), {}),
    ]:
        with pytest.raises(ValueError):
            ops.kv4_paged_decode(*args, **more)
    with pytest.raises(RuntimeError):
        ops.kv4_paged_decode(q, kp.cpu(), vp, tables, ctx, 1.0)
    assert not kp.any() and ops.read_status() == 0


def test_calls_with_nothing_to_do():
    d, bs, h = 64, 16, 2
    kp = torch.zeros((2, h, ops.kv4_page_bytes(bs, d)), dtype=torch.uint8, device="cuda")
    k = torch.zeros((0, h, d), dtype=torch.bfloat16, device="cuda")
    none = torch.zeros(0, dtype=torch.long).cuda()
    ops.kv4_scatter(k, k, None, None, none, kp, kp)
    ops.kv4_store_chunks(k[:, :, None], k[:, :, None], none, none, none.view(0, 1), kp, kp)
    key, value = ops.kv4_gather_blocks(kp, kp, none.view(0, 3), d, torch.bfloat16, lengths=none)
    assert key.shape == (0, 3, bs, h, d)
    key, _ = ops.kv4_gather_blocks(kp, kp, torch.zeros((2, 0), dtype=torch.long).cuda(), d, torch.bfloat16)
    assert key.shape == (2, 0, bs, h, d)
    out = ops.kv4_paged_decode(torch.zeros((0, 4, d), dtype=torch.bfloat16, device="cuda"), kp, kp, none.view(0, 1), none,
                               1.0)
    assert out.shape == (0, 4 * d) and ops.read_status() == 0
