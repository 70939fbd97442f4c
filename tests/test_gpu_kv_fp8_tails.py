"""8-bit decode attention with long tails of tokens whose weights are tiny each and not together.

Bound of an output, with u = half a unit in the last place of its type:
  |err| <= u |want| + A (2^-11 + 2 d) + n 2^-32 max|v|,   A = sum_j p_j |v_j|
2^-11: a probability rounded to fp16, where that is a normal number; below, the rounding is absolute, 2^-25, and the
largest probability is at least 2^7 there, so that it is n 2^-32 max|v| in all; d bounds the error of a score: 128 products
accumulated in fp32, the tensor cores truncating, is at most 128 * 2^-23 of sum_d |q_d k_d| * scale, and it enters both the
numerator and the sum.
"""
import pytest
import torch

from oracle import decode_oracle
from test_gpu_kv_fp8 import F8, HALF_ULP, attend, attn_case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens,q_heads,dtype,splits", [(60001, 4, torch.bfloat16, 0), (60001, 4, torch.float16, 1),
                                                         (60001, 16, torch.bfloat16, 1), (1 << 18, 2, torch.float16, 0),
                                                         (1 << 18, 2, torch.bfloat16, 1), (300000, 16, torch.float16, 3)])
@pytest.mark.parametrize("sink", ["first", "middle", "last"])
def test_a_sink_and_a_tail_of_tiny_weights(sink, tokens, q_heads, dtype, splits):
    """One token with almost all of the weight and a value row of zeros; the others with about 2^-26 of it each and value
    rows of one sign: the output is what the tail adds up to."""
    c = attn_case([tokens], q_heads, 1, 64, dtype, seed=tokens)
    g = torch.Generator().manual_seed(2)
    blocks = c["k_cache"].size(0)
    c["k_scale"].fill_(2.0 ** -7)
    c["v_scale"].fill_(1.0)
    tail = torch.randint(-1, 2, (blocks, 64, 1), generator=g) * 16.0
    k = c["k_cache"].float()
    k[..., 0] = tail
    c["k_cache"] = k.to(F8)
    c["v_cache"] = (torch.rand(c["v_cache"].shape, generator=g) * 200 + 100).to(F8)
    token = {"first": 0, "middle": tokens // 2, "last": tokens - 1}[sink]
    page, row = int(c["table"][0, token // 64]), token % 64
    c["k_cache"][page, row, 0, 0] = 448.0
    c["v_cache"][page, row] = 0.0
    # Dimension 0 alone makes the scores: 26 powers of two between the sink and the tail's middle, 1 more or less around it.
    c["q"].zero_()
    c["q"][..., 0] = 58.25
    got = attend(c, splits)
    want, mag, reach = decode_oracle.paged_attn_fp8_ref(c["q"], c["k_cache"], c["v_cache"], c["k_scale"], c["v_scale"], c["lens"],
                                                        c["table"], c["scale"])
    d = 128 * 2.0 ** -23 * float(reach[0])
    vmax = float(c["v_cache"].float().max())
    bound = (HALF_ULP[dtype] * want.abs() + mag * (2.0 ** -11 + 2 * d) + tokens * 2.0 ** -32 * vmax) * (1 + 2.0 ** -7)
    assert float(want.min()) > 0.1 and float(bound.max()) < 0.1 * float(want.min())
    err = (got.double() - want).abs()
    assert bool((err <= bound).all()), (err / bound).max().item()
