"""Every variant of the few-token expert layer that its launch rules choose, against 64 bits element by element.

Bound of an output element.  Pair p = (t, e) has z = w13[e] x_t (gate g, up u), a = weight silu(g) u, and
A = sum_k |x w|, M = sum over the addends |a w2|:
  dz <= (17/16) H 2^-23 A      a product of 16 terms adds them and the sum so far, each cut off at 2^-23 of the
                               largest of the 17, which is at most A; H / 16 of them follow one another
  da <= weight (|silu'(g)| |u| dg + |silu(g)| du + 1.1 dg du + |u| dg^2 / 4)      |silu'| <= 1.1, |silu''| <= 1/2
  err <= 2^-8 |want| + (1 + 2^-7) (sum |w2| da + M (2^-16 + (17/8 I + 128) 2^-23))
2^-8: the output's rounding to bf16; 2^-16: an activation kept as two bf16 numbers, the second at most 2^-8 of it and
rounded by 2^-8 of itself; 17/8 I: two numbers an activation, otherwise as for dz; 128: SiLU, router and the sums over
warps and CTAs.  Taken over a token's row or over 16 output rows, the rounding of many elements stays under 2^-8 of the
norm, and the rest adds up at random: 2^-8 |want| + 2^-15 |M| in norm.
"""
import pytest
import torch

from electrock_infer_b200 import _C
from oracle import decode_oracle
from test_gpu_few_tokens import DEV, case, run

# Sizes and the variants that they take with 148 SMs: whether a warp of kernel 1 has tiles of its own, rows of a tile of
# kernel 1 in sixteens, CTAs that share a tile of kernel 2.
SIZES = {
    (1, 128, 4744): (True, 1, 1),
    (8, 256, 1192): (True, 1, 1),
    (5, 1024, 1792): (True, 1, 1),
    (32, 256, 2384): (True, 2, 2),
    (32, 256, 2376): (True, 1, 2),
    (8, 1024, 2048): (True, 1, 2),
    (16, 512, 4104): (True, 1, 4),           # a ragged contraction
    (2, 512, 16384): (True, 1, 4),
    (7, 272, 8200): (True, 1, 8),
    (32, 256, 8192): (True, 2, 8),
    (20, 1184, 2056): (False, 1, 2),
    (12, 1088, 4112): (False, 2, 2),
}


def variant(tokens, hidden, inter, sms=148):
    """The launch rules restated."""
    hit = min(2 * tokens, 8)
    rows = 2 if tokens > 8 and inter % 16 == 0 else 1
    alone = -(-hidden // (128 // rows)) <= 8 and hit * inter // (8 * rows) >= 8 * sms
    wide = tokens > 8 and hidden % 32 == 0 and hidden // 32 * 4 >= 3 * sms
    tiles, steps = hidden // (32 if wide else 16), hit * (inter // (64 if wide else 128))
    cluster = 1
    while cluster < 8 and tiles * cluster * 2 <= sms and steps >= 128 * cluster:
        cluster *= 2
    return alone, rows, cluster


def test_the_sizes_reach_every_variant():
    assert {size: variant(*size) for size in SIZES} == SIZES
    taken = set(SIZES.values())
    assert {(a, r) for a, r, _ in taken} >= {(True, 1), (True, 2), (False, 1), (False, 2)}
    assert {c for *_, c in taken} == {1, 2, 4, 8}


def reference(c, renormalize=True):
    """Layer, sum of the addends' sizes and the bound above, all in 64 bits."""
    x, w13, w2 = c["x"].double(), c["w13"].double(), c["w2"].double()
    hidden, inter = x.size(1), w2.size(2)
    want, mag, first = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(x)
    order = torch.argsort(c["logits"].double(), dim=1, descending=True, stable=True)[:, :2]
    weight = torch.softmax(c["logits"].double(), 1).gather(1, order)
    if renormalize:
        weight = weight / weight.sum(1, keepdim=True)
    for e in range(8):
        t, slot = torch.nonzero(order == e, as_tuple=True)
        if t.numel() == 0:
            continue
        w = weight[t, slot][:, None]
        g, u = (x[t] @ w13[e].t()).split(inter, 1)
        dg, du = (x[t].abs() @ w13[e].abs().t() * (17 / 16 * hidden * 2.0 ** -23)).split(inter, 1)
        s = torch.sigmoid(g)
        act = w * g * s * u
        da = w * ((s * (1 + g * (1 - s))).abs() * u.abs() * dg + (g * s).abs() * du + 1.1 * dg * du + u.abs() * dg * dg / 4)
        want[t] += act @ w2[e].t()
        mag[t] += act.abs() @ w2[e].abs().t()
        first[t] += da @ w2[e].abs().t()
    rest = first + mag * (2.0 ** -16 + (17 / 8 * inter + 128) * 2.0 ** -23)
    return want, mag, 2.0 ** -8 * want.abs() + (1 + 2.0 ** -7) * rest


def check(c, got, renormalize=True):
    want, mag, bound = reference(c, renormalize)
    err = (got.double() - want).abs()
    assert torch.isfinite(got.float()).all()
    assert bool((err <= bound).all()), (err / bound).max().item()
    assert bool((err.norm(dim=1) <= 2.0 ** -8 * want.norm(dim=1) + 2.0 ** -15 * mag.norm(dim=1)).all())
    tiles = lambda a: a.view(a.size(0), -1, 16).norm(dim=(0, 2))  # noqa: E731
    assert bool((tiles(err) <= 2.0 ** -8 * tiles(want) + 2.0 ** -15 * tiles(mag)).all())


def test_the_reference_agrees_with_the_oracle():
    c = case(5, 64, 32, seed=1)
    for renormalize in (True, False):
        want, mag, _ = reference(c, renormalize)
        oracle_want, oracle_mag = decode_oracle.few_tokens_ref(c["x"], c["logits"], c["w13"], c["w2"], renormalize)
        assert torch.allclose(want, oracle_want, rtol=1e-12, atol=1e-12) and torch.allclose(mag, oracle_mag, rtol=1e-12)


# The other sizes, shared tiles and one CTA for each tile of kernel 2, with the bound of this file.
SHARED = [(1, 256, 128), (3, 128, 136), (8, 512, 1000), (9, 512, 512), (16, 1024, 256), (32, 1024, 1024), (25, 1040, 72),
          (32, 3584, 136)]


@pytest.mark.gpu
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("tokens,hidden,inter", list(SIZES) + SHARED)
def test_against_64_bits_by_element(tokens, hidden, inter, renormalize):
    c = case(tokens, hidden, inter, seed=tokens + inter)
    check(c, run(c, renormalize), renormalize)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,hidden,inter", [(32, 256, 2384), (32, 256, 2376), (32, 128, 4096), (17, 256, 8192), (29, 512, 4104),
                                                 (32, 1184, 2056)])
def test_all_tokens_on_two_experts(tokens, hidden, inter):
    """Two groups of tokens an expert, in tiles of a warp's own and in tiles that clusters share."""
    c = case(tokens, hidden, inter, seed=tokens)
    c["logits"][:, 3] = 8.0
    c["logits"][:, 6] = 9.0
    c["logits"][tokens // 2, 1] = 20.0
    check(c, run(c))


PATHS = [(8, 256, 1192), (32, 256, 2384), (8, 1024, 2048), (16, 512, 4104), (32, 256, 8192)]


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,hidden,inter", PATHS)
def test_in_place_streams_and_graphs(tokens, hidden, inter):
    c = case(tokens, hidden, inter, seed=5)
    want = run(c)
    d = {k: v.to(DEV) for k, v in c.items()}
    x = d["x"].clone()
    _C.moe_few_tokens(x, x, d["logits"], d["w13"], d["w2"])
    assert torch.equal(x.cpu(), want)
    streams, outs = [torch.cuda.Stream() for _ in range(3)], []
    torch.cuda.synchronize()
    for _ in range(6):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(torch.empty_like(d["x"]))
                _C.moe_few_tokens(outs[-1], d["x"], d["logits"], d["w13"], d["w2"])
    torch.cuda.synchronize()
    assert all(torch.equal(o.cpu(), want) for o in outs)
    graphs, outs = [], []
    for _ in range(2):
        g, o = torch.cuda.CUDAGraph(), torch.zeros_like(d["x"])
        with torch.cuda.graph(g):
            _C.moe_few_tokens(o, d["x"], d["logits"], d["w13"], d["w2"])
        graphs.append(g)
        outs.append(o)
    for _ in range(10):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o.cpu(), want) for o in outs)


@pytest.mark.gpu
@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("tokens,hidden,inter", [(8, 512, 256), (8, 256, 1192), (8, 1024, 2048)])
def test_logits_written_by_a_kernel_that_lets_the_layer_start_early(tokens, hidden, inter, graph):
    """The second kernel reads the logits before its own wait.  Here they are the last rows that a long kernel of this
    library writes, one that lets its successor start while it is still running."""
    c = case(tokens, hidden, inter, seed=5)
    d = {k: v.to(DEV) for k, v in c.items()}
    many = 200000
    g = torch.Generator(device=DEV).manual_seed(3)
    rows = [torch.randn(many, 512, generator=g, device=DEV).to(torch.bfloat16) for _ in range(2)]
    gate = torch.randn(8, 512, generator=g, device=DEV).mul_(512 ** -0.5 * 2).to(torch.bfloat16)
    logits = torch.zeros(many, 8, device=DEV)
    weights, ids = torch.empty(many, 2, device=DEV), torch.empty(many, 2, dtype=torch.int32, device=DEV)
    last = logits[many - tokens:]
    out = torch.empty_like(d["x"])

    def step(x):
        _C.gate_topk_softmax(weights, ids, x, gate, logits_out=logits)
        _C.moe_few_tokens(out, d["x"], last, d["w13"], d["w2"])

    want = []
    for x in rows:
        _C.gate_topk_softmax(weights, ids, x, gate, logits_out=logits)
        torch.cuda.synchronize()
        want.append(run({**c, "logits": last.cpu()}))
    assert not torch.equal(*want)
    calls = [lambda x=x: step(x) for x in rows]
    if graph:
        graphs = [torch.cuda.CUDAGraph() for _ in rows]
        for gr, x in zip(graphs, rows):
            with torch.cuda.graph(gr):
                step(x)
        calls = [gr.replay for gr in graphs]
    got = []
    for i in range(20):
        calls[i % 2]()
        got.append(out.clone())
    torch.cuda.synchronize()
    assert all(torch.equal(o.cpu(), want[i % 2]) for i, o in enumerate(got))
