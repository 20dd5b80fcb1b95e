"""The operators of the 4-bit paged KV cache and of the cache's pages, at the sizes they are used at.

A page of the 4-bit pool is one block of one KV head: ``block_size`` tokens of ``head_dim`` values in
groups of 32 along ``head_dim``.  A group of one token holds 32 codes c in 0..15 and two bfloat16
numbers, its step s and its minimum m, and stands for the values m + s * c:

    m = bf16(min x),  s = bf16((max x - m) / 15),  c = clamp(round((x - m) / s), 0, 15)

(fp32 arithmetic, round to nearest even; c = 0 where s = 0).  The pool is uint8
[num_blocks, num_kv_heads, page bytes]; a page's bytes are the codes [groups, block_size, 16] (byte i
of a group holds value 2i in its low and value 2i + 1 in its high four bits), then the parameters
[block_size, groups, 2] (s, m).  That is 5 bits a value, against 16.

* ``decode``: attention of one query token per sequence over such a cache, through block tables;
* ``append`` / ``chunks``: the store of new tokens (a decode step's one per sequence; a prefill
  step's right-aligned chunks), read back as the values the cache now stands for;
* ``gather``: the history of each sequence as dense pages in the model's type;
* ``copy``: pages copied inside every layer's pools (a fork's private last page, a compaction).
"""

import sys
from pathlib import Path

import numpy as np
import torch

own = False

GROUP = 32
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _ops():
    package = str(Path(__file__).resolve().parents[1] / "mini-infra-qwen3_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    from mini_infra_b200 import ops

    return ops


def listed():
    return [
        # a chat's first answer tokens: one sequence, a prompt of a few words; all latency
        {"name": "decode one short row", "op": "decode", "batch": 1, "hq": 16, "hkv": 8, "dim": 128, "bs": 16,
         "lo": 57, "hi": 57, "type": "bf16"},
        # a decode step of a busy server of the small model, contexts as its benchmark draws them
        {"name": "decode 256 rows to 4096", "op": "decode", "batch": 256, "hq": 16, "hkv": 8, "dim": 128, "bs": 16,
         "lo": 128, "hi": 4096, "type": "bf16"},
        # long contexts at the large model's heads: the case the smaller cache is for
        {"name": "decode 64 rows to 32768", "op": "decode", "batch": 64, "hq": 32, "hkv": 8, "dim": 128, "bs": 16,
         "lo": 1024, "hi": 32768, "type": "bf16"},
        # one long document on one rank of a head partition: few rows, a long axis to split
        {"name": "decode one long row, one head", "op": "decode", "batch": 1, "hq": 8, "hkv": 1, "dim": 128, "bs": 32,
         "lo": 32768, "hi": 32768, "type": "fp16"},
        # short ragged contexts with 64-wide heads, an odd batch
        {"name": "decode 37 rows, 64 wide", "op": "decode", "batch": 37, "hq": 12, "hkv": 6, "dim": 64, "bs": 16,
         "lo": 1, "hi": 333, "type": "fp16"},
        # one decode step's new tokens
        {"name": "append 256 tokens", "op": "append", "batch": 256, "hkv": 8, "dim": 128, "bs": 16, "lo": 1,
         "hi": 4096, "type": "bf16"},
        # one step of a chunked prefill under a budget of 2048 tokens
        {"name": "store 16 chunks of 128", "op": "chunks", "batch": 16, "hkv": 8, "dim": 128, "bs": 16, "lo": 128,
         "hi": 128, "start": 1000, "type": "bf16"},
        # whole prompts of unequal lengths, left-padded to the longest
        {"name": "store 8 prompts to 4096", "op": "chunks", "batch": 8, "hkv": 8, "dim": 128, "bs": 16, "lo": 999,
         "hi": 4096, "start": 0, "type": "fp16"},
        # the second chunk of one prompt reads back its first
        {"name": "gather one history of 333", "op": "gather", "batch": 1, "hkv": 8, "dim": 128, "bs": 16, "lo": 333,
         "hi": 333, "type": "fp16"},
        # the histories of a chunked prefill step over long prompts
        {"name": "gather 16 histories to 16383", "op": "gather", "batch": 16, "hkv": 8, "dim": 128, "bs": 16,
         "lo": 4096, "hi": 16383, "type": "bf16"},
        # three sequences forked: each takes a copy of its last, partly filled page in all layers
        {"name": "fork 3 sequences", "op": "copy", "pairs": 3, "layers": 28, "blocks": 64, "hkv": 8, "dim": 128,
         "bs": 16, "type": "bf16"},
        # a fragmented pool compacted into its lowest pages
        {"name": "compact 512 pages", "op": "copy", "pairs": 512, "layers": 28, "blocks": 1280, "hkv": 8, "dim": 128,
         "bs": 16, "type": "bf16"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def draw(rng):
    limit = max(_cost(c) for c in listed())
    while True:
        op = rng.choice(["decode", "decode", "append", "chunks", "gather", "copy"])
        hq, hkv = rng.choice([(16, 8), (32, 8), (8, 1), (8, 2), (12, 6), (5, 5), (16, 4)])
        case = {"op": op, "hkv": hkv, "dim": rng.choice([64, 128, 128]), "bs": rng.choice([16, 16, 32]),
                "type": rng.choice(["bf16", "fp16"])}
        if op == "copy":
            pairs = _log(rng, 1, 512)
            case.update(pairs=pairs, layers=rng.choice([2, 28, 28]), blocks=2 * pairs + rng.randint(2, 200))
        else:
            hi = _log(rng, 1, {"decode": 32768, "append": 4096, "chunks": 4096, "gather": 16384}[op])
            lo = rng.randint(max(1, hi // 8), hi)
            batch = _log(rng, 1, {"decode": 256, "append": 512, "chunks": 32, "gather": 32}[op])
            case.update(batch=batch, lo=lo, hi=hi)
            if op == "decode":
                case.update(hq=hq)
            if op == "chunks":
                case.update(start=rng.choice([0, rng.randint(1, 2000)]))
            # padded to the longest row, the plain forms hold rows x longest tokens in 32 bits
            if batch * (hi + case.get("start", 0)) > 64 * 32768:
                continue
        if _cost(case) <= limit:
            return case


# ---------------------------------------------------------------------------------------------
# The cache's format, in elementary operations
# ---------------------------------------------------------------------------------------------
def _quantise(x):
    """x [..., D] -> codes uint8 [..., groups, 32], steps and minima bfloat16 [..., groups]."""
    x = x.float().unflatten(-1, (-1, GROUP))
    low = x.amin(-1).bfloat16()
    width = x.amax(-1) - low.float()
    step = (width / torch.full_like(width, 15)).bfloat16()  # a tensor: a scalar's division is a product with its inverse
    wide = step.float().unsqueeze(-1)
    code = torch.where(wide > 0, (x - low.float().unsqueeze(-1)) / wide, torch.zeros_like(x))
    return code.round().clamp(0, 15).to(torch.uint8), step, low


def _views(pool, bs, dim):
    """(codes [N, H, groups, bs, 16], parameter bytes [N, H, bs, groups * 4]) views of a pool."""
    n = dim // GROUP
    return (pool[..., : n * bs * 16].unflatten(-1, (n, bs, 16)), pool[..., n * bs * 16 :].unflatten(-1, (bs, n * 4)))


def _rows(x):
    """Tokens x [..., D] as the bytes a page holds of them: codes [..., groups, 16], parameters [..., groups * 4]."""
    code, step, low = _quantise(x)
    pair = code.unflatten(-1, (16, 2))
    return pair[..., 0] | (pair[..., 1] << 4), torch.stack((step, low), -1).flatten(-2).view(torch.uint8)


def _values(pages, bs, dim):
    """Pages [..., page bytes] -> float32 values [..., bs, D]."""
    n = dim // GROUP
    code = pages[..., : n * bs * 16].unflatten(-1, (n, bs, 16))
    code = torch.stack((code & 15, code >> 4), -1).flatten(-2).transpose(-3, -2)  # [..., bs, groups, 32]
    par = pages[..., n * bs * 16 :].contiguous().view(torch.bfloat16).unflatten(-1, (bs, n, 2)).float()
    return (code * par[..., :1] + par[..., 1:]).flatten(-2)


def _pool(tokens):
    """A pool that holds tokens [N, bs, H, D]."""
    code, par = _rows(tokens)
    n, _, h = code.shape[:3]
    return torch.cat((code.permute(0, 2, 3, 1, 4).reshape(n, h, -1), par.permute(0, 2, 1, 3).reshape(n, h, -1)), -1)


def _pools(g, blocks, bs, hkv, dim):
    """Key and value pools: keys with a mean and a width of their own for each channel, as normed and
    rotated keys have, values around zero."""
    normal = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    key = normal(blocks, bs, hkv, dim).mul_(normal(hkv, dim).abs_().add_(0.3)).add_(normal(hkv, dim))
    key = _pool(key)
    return key, _pool(normal(blocks, bs, hkv, dim))


def _tables(rng, lengths, bs, longest):
    """Block tables over a pool with a tenth of free blocks: (tables [B, width], blocks)."""
    need = -(-lengths // bs)
    blocks = 1 + int(need.sum()) + int(need.sum()) // 10 + 1
    ids = 1 + rng.permutation(blocks - 1)
    tables = np.zeros((len(lengths), -(-longest // bs)), dtype=np.int64)
    held = np.arange(tables.shape[1])[None, :] < need[:, None]
    tables[held] = ids[: int(need.sum())]
    return tables, blocks


def _touched(case):
    """Pages that the longest chunk can touch."""
    return -(-case["hi"] // case["bs"]) + (case["start"] > 0)


def _gpu(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.RandomState(seed % (1 << 31))
    bs, hkv, dim, kind = case["bs"], case["hkv"], case["dim"], TYPES[case["type"]]
    normal = lambda *s: torch.randn(s, generator=g, device="cuda").to(kind)  # noqa: E731
    s = {"case": dict(case), "kind": kind}
    if case["op"] == "copy":
        data = normal(2 * case["layers"], case["blocks"], bs, hkv, dim)
        ids = 1 + rng.permutation(case["blocks"] - 1)[: 2 * case["pairs"]]
        s.update(data=data, pools=list(data.unbind(0)), pairs=_gpu(ids.reshape(-1, 2).astype(np.int64)))
        return s
    b = case["batch"]
    lengths = rng.randint(case["lo"], case["hi"] + 1, size=b).astype(np.int64)
    lengths[rng.randint(b)] = case["hi"]
    start = np.full(b, case.get("start", 0), dtype=np.int64)
    if case["op"] == "chunks":
        start = start + rng.randint(0, 8, size=b) * (case["start"] > 0)
    tables, blocks = _tables(rng, start + lengths, bs, case["hi"] + (case.get("start", 0) + 7 if case.get("start") else 0))
    k_pool, v_pool = _pools(g, blocks, bs, hkv, dim)
    s.update(k_pool=k_pool, v_pool=v_pool, tables=_gpu(tables), lengths=_gpu(lengths))
    if case["op"] == "decode":
        s.update(query=normal(b, case["hq"], dim), scale=dim**-0.5)
    if case["op"] == "append":
        last = (lengths - 1) // bs
        page = tables[np.arange(b), last]
        s.update(key=normal(b, hkv, dim), value=normal(b, hkv, dim), slots=_gpu(page * bs + (lengths - 1) % bs),
                 page=_gpu(page[:, None]), held=_gpu(lengths - last * bs))
    if case["op"] == "chunks":
        width, first = case["hi"], start // bs
        count = -(-(start + lengths) // bs) - first  # the pages a chunk touches, its first one partly filled before
        column = np.arange(_touched(case))[None, :]
        pages = np.take_along_axis(tables, np.minimum(first[:, None] + column, tables.shape[1] - 1), 1)
        pages = pages * (column < count[:, None])
        # the model's layout [B, L, H, D], handed on as [B, H, L, D]
        s.update(key=normal(b, width, hkv, dim).transpose(1, 2), value=normal(b, width, hkv, dim).transpose(1, 2),
                 start=_gpu(start), page=_gpu(pages), held=_gpu(start + lengths - first * bs))
    return s


# ---------------------------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------------------------
def _plain_decode(s):
    c, q = s["case"], s["query"].float()
    b, hkv, dim, bs = c["batch"], c["hkv"], c["dim"], c["bs"]
    q = q.view(b, hkv, c["hq"] // hkv, dim)
    key = _values(s["k_pool"][s["tables"]], bs, dim).transpose(1, 2).flatten(2, 3)  # [B, H, T, D]
    score = q @ key.transpose(-1, -2) * s["scale"]
    del key
    seen = torch.arange(score.shape[-1], device=score.device) < s["lengths"][:, None]
    score = score.masked_fill(~seen[:, None, None, :], float("-inf"))
    p = (score - score.amax(-1, keepdim=True)).exp()
    value = _values(s["v_pool"][s["tables"]], bs, dim).transpose(1, 2).flatten(2, 3)
    return ((p @ value) / p.sum(-1, keepdim=True)).reshape(b, -1).to(s["kind"])


def _plain_gather(s, ids, lengths):
    c = s["case"]
    seen = torch.arange(ids.shape[1] * c["bs"], device=ids.device) < lengths[:, None]
    seen = seen.view(ids.shape[0], ids.shape[1], c["bs"], 1, 1)
    pick = lambda pool: _values(pool[ids], c["bs"], c["dim"]).transpose(2, 3).masked_fill(~seen, 0.0).to(s["kind"])  # noqa: E731
    return pick(s["k_pool"]), pick(s["v_pool"])


def _plain_write(s, pool, tokens, slots):
    """Tokens [T, H, D] into their slots."""
    bs, dim = s["case"]["bs"], s["case"]["dim"]
    codes, pars = _views(pool, bs, dim)
    code, par = _rows(tokens)
    codes[slots // bs, :, :, slots % bs, :] = code
    pars[slots // bs, :, slots % bs, :] = par


def _plain_slots(s):
    """(valid [B, L], slot of every valid token) of right-aligned chunks."""
    bs = s["case"]["bs"]
    width = s["key"].shape[2]
    j = torch.arange(width, device=s["start"].device) - (width - s["lengths"][:, None])
    pos = (s["start"][:, None] + j).clamp(min=0)
    slots = s["tables"].gather(1, pos // bs) * bs + pos % bs
    return j >= 0, slots[j >= 0]


def _plain(s):
    op = s["case"]["op"]
    if op == "decode":
        return _plain_decode(s)
    if op == "gather":
        return _plain_gather(s, s["tables"], s["lengths"])
    if op == "copy":
        s["data"][:, s["pairs"][:, 1]] = s["data"][:, s["pairs"][:, 0]]
        return s["data"]
    if op == "append":
        key, value, slots = s["key"], s["value"], s["slots"]
    else:
        valid, slots = _plain_slots(s)
        key, value = s["key"].transpose(1, 2)[valid], s["value"].transpose(1, 2)[valid]
    _plain_write(s, s["k_pool"], key, slots)
    _plain_write(s, s["v_pool"], value, slots)
    return _plain_gather(s, s["page"], s["held"])


def _own(s):
    ops, op = _ops(), s["case"]["op"]
    if op == "decode":
        return ops.kv4_paged_decode(s["query"], s["k_pool"], s["v_pool"], s["tables"], s["lengths"], s["scale"])
    if op == "copy":
        ops.kv_copy_blocks(s["pools"], s["pairs"])
        return s["data"]
    dim, kind = s["case"]["dim"], s["kind"]
    if op == "gather":
        return ops.kv4_gather_blocks(s["k_pool"], s["v_pool"], s["tables"], dim, kind, lengths=s["lengths"])
    if op == "append":
        ops.kv4_scatter(s["key"], s["value"], None, None, s["slots"], s["k_pool"], s["v_pool"])
    else:
        ops.kv4_store_chunks(s["key"], s["value"], s["lengths"], s["start"], s["tables"], s["k_pool"], s["v_pool"])
    return ops.kv4_gather_blocks(s["k_pool"], s["v_pool"], s["page"], dim, kind, lengths=s["held"])


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    """Each input read once, each output written once.  One row has the longest length, the others count
    their mean."""
    size, bs, hkv, dim = 2, case["bs"], case["hkv"], case["dim"]
    if case["op"] == "copy":
        return {"bytes": 2 * case["pairs"] * 2 * case["layers"] * bs * hkv * dim * size, "flops": 0}
    b = case["batch"]
    tokens = case["hi"] + (b - 1) * (case["lo"] + case["hi"]) / 2
    stored = 2 * hkv * dim * 5 / 8  # bytes of one token's K and V in the cache
    dense = 2 * hkv * dim * size
    if case["op"] == "decode":
        return {"bytes": tokens * (stored + 8 / bs) + 2 * b * case["hq"] * dim * size + 8 * b,
                "flops": 4 * tokens * case["hq"] * dim}
    if case["op"] == "gather":
        padded = b * -(-case["hi"] // bs) * bs
        return {"bytes": tokens * (stored + 8 / bs) + padded * dense, "flops": 2 * tokens * 2 * hkv * dim}
    new = b if case["op"] == "append" else tokens
    back = b * bs if case["op"] == "append" else b * _touched(case) * bs  # the new tokens' pages, as dense ones
    return {"bytes": new * (dense + stored) + new * stored + back * dense, "flops": 8 * new * 2 * hkv * dim}


# ---------------------------------------------------------------------------------------------
# The same from the definitions, in 64 bits
# ---------------------------------------------------------------------------------------------
def _exact_page(pages, bs, dim):
    """Pages [P, H, bytes] -> values [P, bs, H, D] in 64 bits, value by value from their places."""
    d = torch.arange(dim, device=pages.device)
    t = torch.arange(bs, device=pages.device)
    place = ((d // GROUP)[None, :] * bs + t[:, None]) * 16 + (d % GROUP // 2)[None, :]
    code = (pages[:, :, place].long() >> (4 * (d % 2))) & 15
    word = dim // GROUP * bs * 16 + (t[:, None] * (dim // GROUP) + (d // GROUP)[None, :]) * 4
    number = lambda at: ((pages[:, :, at].int() << 16) | (pages[:, :, at + 1].int() << 24)).view(torch.float32).double()  # noqa: E731
    return (number(word + 2) + number(word) * code).transpose(1, 2)


def _exact_stored(x):
    """What the cache stands for after tokens x [..., D] were stored in it."""
    shape, x = x.shape, x.double().reshape(-1, GROUP)
    low = x.min(1, keepdim=True).values.float().bfloat16().double()
    step = ((x.max(1, keepdim=True).values - low) / 15).float().bfloat16().double()
    code = ((x - low) / torch.where(step > 0, step, torch.inf)).round().clamp(0, 15)
    return (low + step * code).reshape(shape)


def exact(case, seed):
    s = prepare(case, seed)
    bs, dim = case["bs"], case["dim"]
    if case["op"] == "copy":
        return None  # no computed numbers
    if case["op"] == "decode":
        out = []
        for b in range(case["batch"]):
            n = int(s["lengths"][b])
            ids = s["tables"][b, : -(-n // bs)]
            key = _exact_page(s["k_pool"][ids], bs, dim).flatten(0, 1)[:n]
            value = _exact_page(s["v_pool"][ids], bs, dim).flatten(0, 1)[:n]
            q = s["query"][b].double().view(case["hkv"], -1, dim)
            p = torch.softmax(torch.einsum("hgd,thd->hgt", q, key) * s["scale"], -1)
            out.append(torch.einsum("hgt,thd->hgd", p, value).reshape(-1))
        return torch.stack(out)
    ids, held = (s["tables"], s["lengths"]) if case["op"] == "gather" else (s["page"], s["held"])
    got = []
    for pool, new in ((s["k_pool"], s.get("key")), (s["v_pool"], s.get("value"))):
        dense = torch.zeros((*ids.shape, bs, case["hkv"], dim), dtype=torch.float64, device="cuda")
        for b in range(case["batch"]):
            n = int(held[b])
            row = _exact_page(pool[ids[b, : -(-n // bs)]], bs, dim).flatten(0, 1)[:n]
            if case["op"] == "append":
                row[n - 1] = _exact_stored(new[b])
            elif case["op"] == "chunks":
                m = int(s["lengths"][b])
                row[n - m :] = _exact_stored(new[b, :, new.shape[2] - m :].transpose(0, 1))
            dense[b].view(-1, case["hkv"], dim)[:n] = row
        got.append(dense)
    return tuple(got)
