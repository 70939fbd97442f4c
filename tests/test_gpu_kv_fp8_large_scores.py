"""8-bit decode attention with scores so large that one token takes everything."""
import pytest
import torch

from test_gpu_kv_fp8 import F8, attend, attn_case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,size,unit", [(torch.bfloat16, 1e4, 2.0 ** -7), (torch.bfloat16, 3e7, 2.0 ** -7),
                                             (torch.bfloat16, 1e10, 2.0 ** -3), (torch.bfloat16, 1e20, 2.0 ** -7),
                                             (torch.float16, 6e4, 2.0 ** 8), (torch.float16, 6e4, 2.0 ** 20)])
@pytest.mark.parametrize("group", [4, 16])
def test_one_token_takes_everything(group, dtype, size, unit):
    """A score that leads by more than any rounding of it: the output is that token's value, however large the scores
    are.  The value is a code times a power of two, which both types hold."""
    c = attn_case([300, 1000], 2 * group, 2, 32, dtype, seed=7)
    g = torch.Generator().manual_seed(1)
    c["q"] = (size * (torch.randint(0, 2, c["q"].shape, generator=g) * 2 - 1)).to(dtype)
    c["k_scale"].fill_(unit)
    c["v_scale"] = torch.exp2(torch.randint(-6, 1, c["v_scale"].shape, generator=g).float())
    for splits in (1, 3, 8):
        for b, first, second in ((0, 5, 290), (1, 700, 999)):
            for kvh, token in ((0, first), (1, second)):
                page, row = int(c["table"][b, token // 32]), token % 32
                head = kvh * group + (first + splits) % group
                c["k_cache"][page, row, kvh] = (448 * torch.sign(c["q"][b, head].float())).to(F8)
        got = attend(c, splits)
        assert torch.isfinite(got.float()).all()
        for b, first, second in ((0, 5, 290), (1, 700, 999)):
            for kvh, token in ((0, first), (1, second)):
                page, row = int(c["table"][b, token // 32]), token % 32
                head = kvh * group + (first + splits) % group
                want = c["v_cache"][page, row, kvh].float() * c["v_scale"][page, kvh]
                assert torch.equal(got[b, head].float(), want)
