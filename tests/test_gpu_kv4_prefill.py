"""Prefill over a 4-bit history: calls on two streams and captured ones share no workspace, tables that are a column
slice, histories of no, some and all columns, against paged_prefill over a dense pool of the same values."""

import pytest
import torch

from mini_infra_b200 import ops

pytestmark = pytest.mark.gpu


def case(seed, b=3, length=160, hq=8, h=2, d=128, bs=16, dtype=torch.bfloat16, starts=(70, 0, 333), width=24):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(s, generator=g, device="cuda").to(dtype)  # noqa: E731
    blocks = b * width + 1
    kp = torch.zeros((blocks, h, ops.kv4_page_bytes(bs, d)), dtype=torch.uint8, device="cuda")
    vp = torch.zeros_like(kp)
    ops.kv4_scatter(rnd(blocks * bs, h, d), rnd(blocks * bs, h, d), None, None, torch.arange(blocks * bs).cuda(), kp, vp)
    tables = 1 + torch.randperm(b * width, generator=g, device="cuda").view(b, width)
    lens = torch.tensor([length, 1, length // 2]).cuda()
    return (rnd(b, length, hq, d), rnd(b, length, h, d), rnd(b, length, h, d), kp, vp, tables, torch.tensor(starts).cuda(),
            lens, d**-0.5)


def over_dense(q, k, v, kp, vp, tables, starts, lens, scale):
    every = torch.arange(kp.shape[0]).cuda()[None]
    key, value = ops.kv4_gather_blocks(kp, vp, every, q.shape[-1], q.dtype)
    return ops.paged_prefill(q, k, v, key[0], value[0], tables, starts, lens, scale)


def assert_close(got, want, q, k, v):
    """Tables of another width may cut the rows' work at other places: two results within the roundings of each.
    16-bit types: half a unit of the output and of every weight; fp32: (n + 64) 2^-24 of the sums, and a score's (2 D + 64)
    2^-24 of |q||k| on every weight, n <= 512; all of at most the largest |v| (4-bit values reach a step past it)."""
    big = v.abs().max().item() * 1.1
    if q.dtype is torch.float32:
        d = q.shape[-1]
        delta = (2 * d + 64) * 2.0**-24 * d**-0.5 * q.norm(dim=-1).max().item() * k.norm(dim=-1).max().item() * 1.5
        tol = torch.full_like(want, (2 * delta + 2 * (512 + 64) * 2.0**-24) * 2 * big)
    else:
        tol = 2 * torch.finfo(q.dtype).eps / 2 * (want.float().abs() + big) * 1.01
    assert ((got.float() - want.float()).abs() <= tol).all()


@pytest.mark.parametrize("kind", [dict(), dict(dtype=torch.float16, hq=4, h=4), dict(dtype=torch.float32, d=32, bs=3, length=40),
                                  dict(d=64, bs=32)])
def test_over_the_history_it_copies(kind):
    args = case(1, **kind)
    q, tables, starts = args[0], args[5], args[6]
    need = int(-(-starts.max() // (args[3].shape[2] // (q.shape[-1] * 5 // 8))))
    if q.dtype is torch.float32:
        starts.clamp_(max=70)
        need = 24
    want = over_dense(*args)
    assert torch.equal(ops.kv4_paged_prefill(*args), want)
    assert_close(ops.kv4_paged_prefill(*args[:5], tables[:, :need], *args[6:]), want, *args[:3])
    starts.zero_()
    want = ops.paged_prefill(*args[:3], None, None, tables[:, :0], *args[6:])
    assert torch.equal(ops.kv4_paged_prefill(*args[:5], tables[:, :0], *args[6:]), want)
    assert_close(ops.kv4_paged_prefill(*args), want, *args[:3])
    assert ops.read_status() == 0


def test_two_streams_and_a_captured_graph_share_no_workspace(monkeypatch):
    """Rows cut over many CTAs, so that every call keeps partial sums in its workspace."""
    args = [case(seed, length=192, starts=(5000, 3000, 4000), width=400) for seed in (1, 2)]
    want = [over_dense(*x) for x in args]
    torch.cuda.synchronize()

    def shared(*_, **__):
        raise AssertionError("the device's shared workspace")

    monkeypatch.setattr(ops, "workspace", shared)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(10):
        got = []
        for s, x in zip(streams, args):
            with torch.cuda.stream(s):
                got.append(ops.kv4_paged_prefill(*x))
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graphs, outs = [], []
    for x in args:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(ops.kv4_paged_prefill(*x))
        graphs.append(graph)
    for _ in range(5):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        again = ops.kv4_paged_prefill(*args[0])
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]) and torch.equal(again, want[0])
    assert ops.read_status() == 0


def test_workspaces_of_another_form_are_refused():
    q, k, v, kp, vp, tables, starts, lens, scale = case(1)
    starts.zero_()
    args = (q, k, v, None, None, tables[:, :0], starts, lens, scale)
    with pytest.raises(ValueError, match="ws"):
        ops.paged_prefill(*args, ws=torch.zeros(1 << 27, dtype=torch.uint8, device="cuda")[::2])
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        ops.paged_prefill(*args, ws=torch.zeros(1 << 20, dtype=torch.uint8))
    with pytest.raises(ValueError, match="workspace"):
        ops.paged_prefill(*args, ws=torch.zeros(512, dtype=torch.uint8, device="cuda"))
    want = ops.paged_prefill(*args)
    assert torch.equal(ops.paged_prefill(*args, ws=torch.zeros(1 << 27, dtype=torch.uint8, device="cuda")), want)
