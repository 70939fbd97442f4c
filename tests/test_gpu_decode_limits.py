"""Decode-step operators at the ends of their documented ranges."""
import pytest
import torch

from electrock_infer_b200 import _C
from test_gpu_kv_fp8 import attn_case

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("rows", [2 ** 31 - 6, 2 ** 31 - 4, 2 ** 31 - 2])
def test_schedule_with_as_many_rows_as_it_takes(rows):
    """The largest slot map of a call: live rows at its beginning, everything behind them marked."""
    i32 = dict(dtype=torch.int32, device=DEV)
    lens, new = torch.tensor([5, 40, 7], **i32), torch.tensor([3, -1, 60], **i32)
    table = torch.tensor([[2, -1, -1, -1, -1], [0, 1, 4, -1, -1], [3, -1, -1, -1, -1]], **i32)
    free, count = torch.tensor([9, 8, -7, -7, -7], **i32), torch.tensor([2], **i32)
    seq, cu = torch.zeros(3, **i32), torch.full((4,), -5, **i32)
    left, refused = torch.full((1,), -5, **i32), torch.full((1,), -5, **i32)
    slots = torch.zeros(rows, **i32)
    _C.paged_schedule(lens, new, table, free, count, 16, seq, cu, slots, None, left, refused)
    torch.cuda.synchronize()
    assert seq.tolist() == [8, 0, 67] and cu.tolist() == [0, 3, 3, 63] and refused.tolist() == [0] and left.tolist() == [1]
    # The ended request's pages 0, 1, 4 are pushed on 9, 8; the third pops 4, 1, 0, 8.
    assert table[2].tolist() == [3, 4, 1, 0, 8]
    pages = [3, 4, 1, 0, 8]
    want = [2 * 16 + p for p in range(5, 8)] + [pages[p // 16] * 16 + p % 16 for p in range(7, 67)]
    assert slots[:63].tolist() == want
    for part in slots[63:].split(1 << 28):
        assert int(part.max()) == -1 == int(part.min())


@pytest.mark.parametrize("splits", [65, 10 ** 6, 2 ** 31 - 1])
def test_attention_refuses_too_many_splits_before_it_allocates_their_scratch(splits):
    c = attn_case([10, 20], 32, 8, 32, torch.bfloat16, seed=1)
    d = {k: (v.to(DEV) if torch.is_tensor(v) else v) for k, v in c.items()}
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    with pytest.raises(RuntimeError, match="num_splits"):
        _C.paged_attn_varlen_fp8(d["q"], d["k_cache"], d["v_cache"], d["k_scale"], d["v_scale"], 0, d["lens"], d["table"], 0.1,
                                 num_splits=splits)
    assert torch.cuda.max_memory_allocated() - before <= 2 * 32 * 128 * 2      # the output
