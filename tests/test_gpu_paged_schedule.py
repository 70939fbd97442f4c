"""Step tables built on the GPU against a request-by-request restatement: integer outputs, equal."""
import numpy as np
import pytest
import torch

from electrock_infer_b200 import _C
from oracle import decode_oracle

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def make(ctx, new, block_size, width, spare, seed, rows=None, capacity=None, stride=None):
    """Requests with pages dealt out at random, `spare` free pages and a table `width` pages wide."""
    rng = np.random.default_rng(seed)
    ctx, new = np.asarray(ctx), np.asarray(new)
    have = [min(-(-max(int(c), 0) // block_size), width) for c in ctx]
    pool = sum(have) + spare
    order = rng.permutation(pool)
    table = np.full((len(ctx), width), -1, np.int64)
    at = 0
    for i, n in enumerate(have):
        table[i, :n] = order[at:at + n]
        at += n
    free = np.full(pool if capacity is None else capacity, -7, np.int64)
    free[:spare] = order[at:]
    total = int(np.maximum(new, 0).sum())
    return {"ctx": ctx, "new": new, "table": table, "free": free, "count": spare, "bs": block_size,
            "rows": total if rows is None else rows, "stride": stride or width}


def i32(a):
    return torch.as_tensor(np.asarray(a), dtype=torch.int32, device=DEV)


def run(c, alias=False, positions=True, offset=0):
    n = len(c["ctx"])
    wide = torch.full((max(n, 1), c["stride"]), 12345, dtype=torch.int32, device=DEV)
    table = wide[:n, : c["table"].shape[1]]
    table.copy_(i32(c["table"]))
    d = {"context_lens": i32(c["ctx"]), "free_blocks": i32(c["free"]), "free_count": i32([c["count"]]), "block_table": table}
    d["seq_lens"] = d["context_lens"] if alias else torch.full((n,), -5, dtype=torch.int32, device=DEV)
    d["free_count_out"] = d["free_count"] if alias else i32([-5])
    d["cu_seqlens"] = torch.full((n + 1,), -5, dtype=torch.int32, device=DEV)
    d["num_refused"] = i32([-5])
    d["slot_mapping"] = torch.full((c["rows"] + offset,), -5, dtype=torch.int32, device=DEV)[offset:]
    d["positions"] = torch.full((c["rows"] + offset,), -5, dtype=torch.int64, device=DEV)[offset:] if positions else None
    _C.paged_schedule(d["context_lens"], i32(c["new"]), table, d["free_blocks"], d["free_count"], c["bs"], d["seq_lens"],
                      d["cu_seqlens"], d["slot_mapping"], d["positions"], d["free_count_out"], d["num_refused"])
    torch.cuda.synchronize()
    if c["stride"] > c["table"].shape[1]:
        assert bool((wide[:, c["table"].shape[1]:] == 12345).all())
    return d


def same(c, d):
    want = decode_oracle.paged_schedule_ref(c["ctx"], c["new"], c["table"], c["free"], c["count"], c["bs"], c["rows"])
    for key in ("block_table", "free_blocks", "seq_lens", "cu_seqlens", "slot_mapping"):
        assert np.array_equal(d[key].cpu().numpy(), want[key]), key
    if d["positions"] is not None:
        assert np.array_equal(d["positions"].cpu().numpy(), want["positions"])
    assert int(d["free_count_out"]) == want["free_count_out"] and int(d["num_refused"]) == want["num_refused"]
    return want


CASES = {
    "one token": dict(ctx=[0], new=[1], block_size=256, width=1, spare=1),
    "decode": dict(ctx=[5, 256, 255, 1000, 0], new=[1] * 5, block_size=256, width=8, spare=9),
    "page edges": dict(ctx=[15, 16, 17, 0, 31, 32], new=[1, 1, 1, 16, 2, 17], block_size=16, width=5, spare=20),
    "prompts": dict(ctx=[0, 3, 700], new=[1234, 55, 1], block_size=48, width=40, spare=64),
    "ended and waiting": dict(ctx=[40, 33, 0, 100, 7], new=[-1, 0, -3, 20, -1], block_size=16, width=10, spare=0),
    "pops released pages": dict(ctx=[64, 0, 48], new=[-1, 100, -9], block_size=16, width=8, spare=1),
    "out of pages": dict(ctx=[0, 0, 10, 0, 16], new=[32, 33, 1, 1, 0], block_size=16, width=8, spare=3),
    "first too large": dict(ctx=[0, 0], new=[100, 1], block_size=16, width=8, spare=3),
    "row too short": dict(ctx=[120, 5], new=[20, 4], block_size=16, width=8, spare=9),
    "few rows": dict(ctx=[4, 4, 4, 4], new=[3, 3, 3, 3], block_size=16, width=2, spare=4, rows=8),
    "padded rows": dict(ctx=[4, 9], new=[3, 2], block_size=4, width=4, spare=4, rows=70),
    "nobody": dict(ctx=[9, 9], new=[0, -1], block_size=4, width=4, spare=0, rows=16),
    "no rows": dict(ctx=[9, 9], new=[0, -1], block_size=4, width=4, spare=2, rows=0),
    "length beyond the row": dict(ctx=[1000, -4, 2 ** 31 - 1], new=[-1, 3, 1], block_size=4, width=4, spare=2),
    "page of one": dict(ctx=[3, 0, 2], new=[2, 4, -1], block_size=1, width=6, spare=5),
    "small stack": dict(ctx=[64, 64], new=[-1, -1], block_size=16, width=4, spare=2, capacity=7),
    "huge request": dict(ctx=[10, 10], new=[2 ** 31 - 1, 2 ** 31 - 1], block_size=16, width=4, spare=2, rows=5),
    "strided table": dict(ctx=[15, 40, 3], new=[2, 30, -1], block_size=16, width=6, spare=20, stride=11),
}


@pytest.mark.parametrize("alias", [False, True])
@pytest.mark.parametrize("name", list(CASES))
def test_small_steps(name, alias):
    c = make(seed=len(name), **CASES[name])
    same(c, run(c, alias))


@pytest.mark.parametrize("requests,most,block_size,spare,pad", [
    (1, 5000, 16, 400, 3), (7, 900, 32, 150, 0), (257, 60, 16, 900, 1), (1000, 9, 256, 1200, 96),
    (4099, 1, 16, 700, 5), (8192, 3, 64, 9000, 17), (33, 4000, 128, 600, 0)])
def test_ragged_steps(requests, most, block_size, spare, pad):
    rng = np.random.default_rng(requests + most)
    ctx = rng.integers(0, 3 * block_size, requests)
    new = rng.integers(1, most + 1, requests)
    kind = rng.random(requests)
    new[(kind < 0.1) & (requests > 1)] = -1
    new[(kind > 0.9) & (requests > 1)] = 0
    width = 3 + most // block_size + 1
    c = make(ctx, new, block_size, width, spare, seed=3, rows=int(np.maximum(new, 0).sum()) + pad)
    same(c, run(c))
    same(c, run(c, alias=True, positions=False))


def test_outputs_without_16_byte_alignment():
    c = make([3, 100, 0], [50, 1, 70], 16, 12, 30, seed=5)
    for offset in (1, 2, 3):
        same(c, run(c, offset=offset))


def test_no_requests():
    c = make([], [], 16, 4, 3, seed=1, rows=9)
    d = run(c)
    assert d["cu_seqlens"].tolist() == [0] and int(d["free_count_out"]) == 3
    assert d["slot_mapping"].tolist() == [-1] * 9 and d["positions"].tolist() == [0] * 9


def test_steps_follow_one_another_in_place():
    """Forty decode steps with requests that end and restart, lengths and stack updated in place: every
    page belongs to one request or to the stack at all times."""
    rng = np.random.default_rng(11)
    n, bs, width, pool = 24, 16, 9, 120
    lens = torch.zeros(n, dtype=torch.int32, device=DEV)
    table = torch.full((n, width), -1, dtype=torch.int32, device=DEV)
    free = torch.arange(pool, dtype=torch.int32, device=DEV).flip(0).contiguous()
    count, refused = i32([pool]), i32([0])
    cu = torch.empty(n + 1, dtype=torch.int32, device=DEV)
    for step in range(40):
        new = rng.integers(1, 12, n)
        new[rng.random(n) < 0.15] = -1
        new[rng.random(n) < 0.1] = 0
        rows = int(np.maximum(new, 0).sum()) + 5
        slots = torch.empty(rows, dtype=torch.int32, device=DEV)
        pos = torch.empty(rows, dtype=torch.int64, device=DEV)
        want = decode_oracle.paged_schedule_ref(lens.tolist(), new, table.cpu().numpy(), free.cpu().numpy(), int(count), bs, rows)
        _C.paged_schedule(lens, i32(new), table, free, count, bs, lens, cu, slots, pos, count, refused)
        assert np.array_equal(slots.cpu().numpy(), want["slot_mapping"])
        assert lens.tolist() == want["seq_lens"].tolist() and int(count) == want["free_count_out"]
        held = [int(p) for i in range(n) for p in table[i, : -(-int(lens[i]) // bs)]]
        assert sorted(held + free[: int(count)].tolist()) == list(range(pool))


def test_side_stream_and_graph():
    c = make([3, 100, 0, 31], [5, 1, 70, -1], 16, 12, 30, seed=5)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        d = run(c)
    same(c, d)
    new = i32(c["new"])
    args = (d["context_lens"], new, d["block_table"], d["free_blocks"], d["free_count"], c["bs"], d["seq_lens"],
            d["cu_seqlens"], d["slot_mapping"], d["positions"], d["free_count_out"], d["num_refused"])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        _C.paged_schedule(*args)
    c2 = make([30, 1, 16, 0], [1, 75, 0, -1], 16, 12, 30, seed=6, rows=c["rows"])
    d["context_lens"].copy_(i32(c2["ctx"]))
    new.copy_(i32(c2["new"]))
    d["block_table"].copy_(i32(c2["table"]))
    full = torch.full_like(d["free_blocks"], -7)
    full[: len(c2["free"])] = i32(c2["free"])[: full.numel()]
    d["free_blocks"].copy_(full)
    c2["free"] = full.cpu().numpy()
    g.replay()
    torch.cuda.synchronize()
    same(c2, d)


def test_refusals():
    c = make([3, 4], [1, 1], 16, 4, 4, seed=1)
    d = run(c)
    new = i32(c["new"])

    def call(**kw):
        a = {**d, "new_lens": new, "block_size": 16, **kw}
        _C.paged_schedule(a["context_lens"], a["new_lens"], a["block_table"], a["free_blocks"], a["free_count"],
                          a["block_size"], a["seq_lens"], a["cu_seqlens"], a["slot_mapping"], a["positions"],
                          a["free_count_out"], a["num_refused"])

    call()
    for bad in (dict(context_lens=d["context_lens"].long()), dict(new_lens=new[:1]), dict(block_size=0),
                dict(block_table=d["block_table"].long()), dict(block_table=d["block_table"].t()),
                dict(cu_seqlens=d["seq_lens"]), dict(positions=d["positions"].int()),
                dict(positions=d["positions"][:1]), dict(free_count=d["seq_lens"]), dict(slot_mapping=d["slot_mapping"].cpu()),
                dict(block_size=2 ** 30), dict(block_table=d["block_table"][:, :0])):
        with pytest.raises(RuntimeError):
            call(**bad)
    many = _C.paged_schedule_max_requests() + 1
    z = torch.zeros(many, dtype=torch.int32, device=DEV)
    with pytest.raises(RuntimeError, match="at most"):
        call(context_lens=z, new_lens=z, seq_lens=z.clone(), cu_seqlens=torch.zeros(many + 1, dtype=torch.int32, device=DEV),
             block_table=torch.zeros(many, 2, dtype=torch.int32, device=DEV))
