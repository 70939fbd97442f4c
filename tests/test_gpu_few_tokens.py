"""The few-token expert layer against the definition in 64 bits.

Bound of an output element, with M = sum over its addends |w act w2|:
  |err| <= 2^-8 |want| + M (2^-16 + (I + H + 64) 2^-23 + r)
2^-8: the output's rounding to bf16; 2^-16: an activation kept as two bf16 numbers (the rest after the
first, at most 2^-8 of it, is rounded by at most 2^-8 of itself; times 1 for the sum); (I + H + 64) 2^-23:
fp32 accumulation over the two contractions (truncating tensor cores), the router and the SiLU; r: the
first contraction's error relative to its addends, which cancel: 2^-23 H sum|x w| / |x w|, seen through
silu(gate) * up it is taken from the data as H 2^-23 times the ratio of the largest sum|x w| to the typical
activation (computed below).
"""
import pytest
import torch

from electrock_infer_b200 import _C, _lib
from electrock_infer_b200.layers.moe import FusedMoE, fused_experts
from electrock_infer_b200.layers.moe.mixtral_moe import MixtralMoE
from oracle import decode_oracle

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def case(tokens, hidden, inter, seed, logits_dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    return {"x": rand(tokens, hidden).to(torch.bfloat16), "logits": (rand(tokens, 8) * 1.5).to(logits_dtype),
            "w13": (rand(8, 2 * inter, hidden) * hidden ** -0.5).to(torch.bfloat16),
            "w2": (rand(8, hidden, inter) * inter ** -0.5).to(torch.bfloat16)}


def run(c, renormalize=True, out=None):
    d = {k: v.to(DEV) for k, v in c.items()}
    out = torch.full_like(d["x"], 7.0) if out is None else out
    _C.moe_few_tokens(out, d["x"], d["logits"], d["w13"], d["w2"], renormalize=renormalize)
    torch.cuda.synchronize()
    return out.cpu()


def bound(c, want, mag):
    hidden, inter = c["w13"].size(2), c["w2"].size(2)
    # First contraction: |x . w| is about 1 by construction, sum|x w| at most this.
    reach = (c["x"].float().abs().amax(0).double() @ c["w13"].float().abs().amax((0, 1)).double()).item()
    first = hidden * 2.0 ** -23 * reach * 2 * c["w2"].float().abs().sum(-1).amax().double()
    return (2.0 ** -8 * want.abs() + mag * (2.0 ** -16 + (inter + hidden + 64) * 2.0 ** -23)) * (1 + 2.0 ** -7) + first


def check(c, got, renormalize=True):
    want, mag = decode_oracle.few_tokens_ref(c["x"], c["logits"], c["w13"], c["w2"], renormalize)
    err = (got.double() - want).abs()
    assert torch.isfinite(got.float()).all()
    assert bool((err <= bound(c, want, mag)).all()), (err - bound(c, want, mag)).max().item()
    # The bound above is loose for single elements; as a whole the result is as good as its rounding.
    assert err.norm() <= 2.0 ** -8 * want.norm()


@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("tokens,hidden,inter", [
    (1, 256, 128), (1, 16, 8), (2, 48, 24), (3, 128, 136), (7, 336, 288), (8, 512, 1000), (9, 512, 512), (15, 272, 776),
    (16, 1024, 256), (17, 256, 512), (24, 144, 64), (25, 512, 264), (31, 640, 128), (32, 1024, 1024)])
def test_against_64_bits(tokens, hidden, inter, renormalize):
    c = case(tokens, hidden, inter, seed=tokens + hidden)
    check(c, run(c, renormalize), renormalize)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_logit_types(dtype):
    c = case(13, 256, 128, seed=4, logits_dtype=dtype)
    check(c, run(c))


def test_at_full_hidden_size():
    c = case(5, 4096, 1792, seed=2)
    check(c, run(c))


def test_ties_and_masked_logits():
    """Equal logits take the lower index; -inf and the lowest finite value are ordinary logits; one expert
    may get all tokens, others none."""
    c = case(12, 256, 128, seed=6)
    low = torch.finfo(torch.float32).min
    c["logits"][0] = 1.0
    c["logits"][1] = torch.tensor([0., 3, 3, 3, 0, 0, 0, 0])
    c["logits"][2] = torch.tensor([low] * 7 + [2.0])
    c["logits"][3] = torch.tensor([-torch.inf] * 5 + [1.0, 0.5, -torch.inf])
    c["logits"][4:] = torch.tensor([0., 0, 0, 0, 9, 0, 0, 8])
    check(c, run(c))
    c["logits"][5] = torch.tensor([-torch.inf] * 3 + [1.0] + [-torch.inf] * 4)   # the second has weight 0
    got = run(c)
    d = {k: v[5:6] if k in ("x", "logits") else v for k, v in c.items()}
    z = d["w13"][3].double() @ d["x"][0].double()
    act = z[:128] / (1 + torch.exp(-z[:128])) * z[128:]
    assert (got[5].double() - d["w2"][3].double() @ act).norm() <= 2.0 ** -8 * (d["w2"][3].double() @ act).norm()


@pytest.mark.parametrize("tokens,hidden,inter", [(17, 256, 128), (32, 4096, 256), (32, 512, 1000), (32, 2400, 520), (25, 1040, 72)])
def test_all_tokens_on_two_experts(tokens, hidden, inter):
    """More tokens of an expert than a ring stage holds: its weights are gone through twice."""
    c = case(tokens, hidden, inter, seed=tokens)
    c["logits"][:, 3] = 8.0
    c["logits"][:, 6] = 9.0
    c["logits"][tokens // 2, 1] = 20.0
    check(c, run(c))


def test_large_and_saturated_gates():
    c = case(6, 256, 128, seed=8)
    c["x"] *= 60
    got = run(c)
    want, _ = decode_oracle.few_tokens_ref(c["x"], c["logits"], c["w13"], c["w2"])
    assert torch.isfinite(got.float()).all() and (got.double() - want).norm() <= 2.0 ** -8 * want.norm()


def test_activations_beyond_the_range_become_infinities():
    """An activation that overflows is an infinity, as in fp32, and does not turn into NaN on its way; other tokens
    are not touched."""
    c = case(3, 32, 16, seed=2)
    c["w13"].zero_()
    c["w13"][:, 0, 0] = c["w13"][:, 16, 0] = 1.0        # gate and up of element 0 are x[0]
    c["w2"].zero_()
    c["w2"][:, :, 0] = 1.0
    c["w2"][:, 1, 0] = -1.0
    c["x"][0, 0], c["x"][1, 0], c["x"][2, 0] = 1e25, 2.0, 1.85e19
    got = run(c).float()
    assert got[0, 0] == torch.inf and got[0, 1] == -torch.inf and not torch.isnan(got).any()
    assert torch.isfinite(got[1]).all() and abs(got[1, 0].item() - 2 * 2 / (1 + 2.718281828 ** -2)) < 2 ** -8 * 4


def test_in_place_and_no_tokens():
    c = case(9, 512, 256, seed=3)
    want = run(c)
    d = {k: v.to(DEV) for k, v in c.items()}
    _C.moe_few_tokens(d["x"], d["x"], d["logits"], d["w13"], d["w2"])
    assert torch.equal(d["x"].cpu(), want)
    empty = torch.empty(0, 512, dtype=torch.bfloat16, device=DEV)
    _C.moe_few_tokens(empty, empty, torch.empty(0, 8, device=DEV), d["w13"], d["w2"])


def test_rows_behind_the_batch_stay():
    c = case(5, 256, 128, seed=3)
    wide = torch.full((9, 256), 3.0, dtype=torch.bfloat16, device=DEV)
    run(c, out=wide[:5])
    assert bool((wide[5:] == 3).all()) and not bool((wide[:5] == 3).all())


def test_same_bits_every_time_on_streams_and_in_graphs():
    c = case(11, 1024, 512, seed=5)
    want = run(c)
    d = {k: v.to(DEV) for k, v in c.items()}
    outs = []
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for _ in range(6):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(torch.empty_like(d["x"]))
                _C.moe_few_tokens(outs[-1], d["x"], d["logits"], d["w13"], d["w2"])
    torch.cuda.synchronize()
    assert all(torch.equal(o.cpu(), want) for o in outs)
    # Two graphs captured one after the other, replayed at the same time.
    graphs, gouts = [], []
    for _ in range(2):
        g, o = torch.cuda.CUDAGraph(), torch.zeros_like(d["x"])
        with torch.cuda.graph(g):
            _C.moe_few_tokens(o, d["x"], d["logits"], d["w13"], d["w2"])
        graphs.append(g)
        gouts.append(o)
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o.cpu(), want) for o in gouts)


def test_logits_written_right_before_the_call():
    """The second kernel reads the logits before the first has finished: they must be those of the step."""
    c = case(8, 512, 256, seed=5)
    d = {k: v.to(DEV) for k, v in c.items()}
    alt = d["logits"].flip(1).contiguous()
    a, b = run(c), run({**c, "logits": c["logits"].flip(1).contiguous()})
    logits, out = d["logits"].clone(), torch.empty_like(d["x"])
    got = []
    for i in range(40):
        logits.copy_(alt if i % 2 else d["logits"])
        _C.moe_few_tokens(out, d["x"], logits, d["w13"], d["w2"])
        got.append(out.clone())
    torch.cuda.synchronize()
    assert all(torch.equal(o.cpu(), b if i % 2 else a) for i, o in enumerate(got))


def test_through_the_layers():
    c = case(6, 512, 256, seed=9)
    want = run(c)
    d = {k: v.to(DEV) for k, v in c.items()}
    assert torch.equal(fused_experts(d["x"], d["w13"], d["w2"], d["logits"], 2, few_tokens=True).cpu(), want)
    general = fused_experts(d["x"], d["w13"], d["w2"], d["logits"], 2).cpu()
    assert (general.double() - want.double()).norm() <= 2.0 ** -6 * want.double().norm()
    half = fused_experts(d["x"].half(), d["w13"], d["w2"], d["logits"], 2, few_tokens=True)
    assert half.dtype == torch.float16
    layer = FusedMoE(8, 2, 512, 256, params_dtype=torch.bfloat16, few_token_limit=6).to(DEV)
    layer.w13_weight.data.copy_(d["w13"])
    layer.w2_weight.data.copy_(d["w2"])
    x = d["x"].clone()
    assert torch.equal(layer(x, d["logits"]).cpu(), want) and torch.equal(x.cpu(), want)
    seven = case(7, 512, 256, seed=10)
    x7 = seven["x"].to(DEV)
    assert torch.equal(layer(x7.clone(), seven["logits"].to(DEV)),
                       fused_experts(x7, d["w13"], d["w2"], seven["logits"].to(DEV), 2))
    block = MixtralMoE(8, 2, 512, 256, params_dtype=torch.bfloat16, few_token_limit=8).to(DEV)
    block.gate.weight.data.normal_()
    block.experts.w13_weight.data.copy_(d["w13"])
    block.experts.w2_weight.data.copy_(d["w2"])
    got = block(d["x"].clone())
    logits = block.gate(d["x"])
    assert torch.equal(got, fused_experts(d["x"], d["w13"], d["w2"], logits, 2, few_tokens=True))


def test_refusals():
    c = case(4, 256, 128, seed=1)
    d = {k: v.to(DEV) for k, v in c.items()}
    ok = dict(output=torch.empty_like(d["x"]), hidden_states=d["x"], gating_output=d["logits"], w13=d["w13"], w2=d["w2"])
    _C.moe_few_tokens(**ok)
    big = torch.zeros(33, 256, dtype=torch.bfloat16, device=DEV)
    for bad in (dict(hidden_states=d["x"].half()), dict(output=ok["output"][:3]), dict(gating_output=d["logits"][:, :7].contiguous()),
                dict(gating_output=d["logits"].double()), dict(w13=d["w13"][:, :-2].contiguous()), dict(w2=d["w2"].transpose(1, 2)),
                dict(w13=d["w13"].cpu()), dict(w13=d["w13"][:7].contiguous(), w2=d["w2"][:7].contiguous(), gating_output=d["logits"][:, :7].contiguous()),
                dict(hidden_states=big, output=big, gating_output=torch.zeros(33, 8, device=DEV))):
        with pytest.raises(RuntimeError):
            _C.moe_few_tokens(**{**ok, **bad})
    with pytest.raises(RuntimeError):
        fused_experts(d["x"], d["w13"], d["w2"], None, 2, gate_weight=torch.zeros(8, 256, dtype=torch.bfloat16, device=DEV), few_tokens=True)
    rc = _lib.load().b200moe_few_tokens(d["x"].data_ptr(), d["logits"].data_ptr(), _lib.F32, d["w13"].data_ptr(), d["w2"].data_ptr(),
                                        d["x"].data_ptr(), 4, 8, 2, 256, 128, 1, None, 0, torch.cuda.current_stream().cuda_stream)
    assert rc == -4
