"""Decode-step operators without a GPU: argument checks of the C entries and of the Python ops, the
choices made on the host, and the oracle against independent arithmetic."""
import ctypes

import numpy as np
import pytest
import torch

from electrock_infer_b200 import _C, _lib
from oracle import decode_oracle

PTR = ctypes.c_void_p(256)  # never dereferenced: validation fails first


def test_schedule_arguments():
    lib = _lib.load()

    def call(requests=4, width=8, stride=8, block=16, room=32, rows=4, ctx=PTR, slots=PTR, count=PTR):
        return lib.b200moe_paged_schedule(ctx, PTR, PTR, PTR, count, requests, width, stride, block, room, rows, PTR, PTR, slots,
                                          PTR, PTR, PTR, None)

    assert lib.b200moe_paged_schedule_max_requests() == 8192
    for bad in (dict(requests=8193), dict(requests=-1), dict(width=0), dict(stride=7), dict(block=0), dict(width=2 ** 27, stride=2 ** 27),
                dict(room=-1), dict(rows=-1), dict(rows=2 ** 31 - 1), dict(room=2 ** 31)):
        assert call(**bad) == -1, bad
    for bad in (dict(ctx=None), dict(slots=None), dict(count=None)):
        assert call(**bad) == -3, bad


def test_store_arguments():
    lib = _lib.load()

    def call(dtype=_lib.BF16, tokens=4, heads=2, dim=128, ks=256, vs=256, blocks=4, block=16, key=PTR, scale=PTR):
        return lib.b200moe_paged_store_kvcache_fp8(key, PTR, PTR, PTR, scale, PTR, PTR, dtype, tokens, heads, dim, ks, vs, blocks,
                                                   block, None)

    for bad in (dict(dim=64), dict(tokens=-1), dict(heads=0), dict(blocks=-1), dict(block=0), dict(ks=255), dict(vs=128)):
        assert call(**bad) == -1, bad
    assert call(dtype=5) == -2
    assert call(key=None) == -3 and call(scale=None) == -3
    assert call(ks=260) == -5 and call(key=ctypes.c_void_p(264)) == -5
    assert call(tokens=0) == 0


def test_attention_arguments():
    lib = _lib.load()

    def call(dtype=_lib.BF16, batch=2, heads=8, kv=2, dim=128, qs=1024, blocks=4, block=16, width=3, ts=3, splits=1, q=PTR, ws=None,
             ws_bytes=0, scale=PTR):
        return lib.b200moe_paged_attn_varlen_fp8(q, PTR, PTR, scale, PTR, PTR, PTR, PTR, dtype, batch, heads, kv, dim, qs, blocks, block,
                                                 width, ts, 0.1, splits, ws, ws_bytes, None)

    for bad in (dict(dim=64), dict(heads=7), dict(kv=0), dict(batch=-1), dict(block=8), dict(block=24), dict(blocks=0), dict(width=0),
                dict(ts=2), dict(splits=0), dict(splits=65), dict(qs=1000)):
        assert call(**bad) == -1, bad
    assert call(dtype=_lib.F32) == -2
    assert call(heads=34, qs=34 * 128) == -7
    assert call(q=None) == -3 and call(scale=None) == -3
    assert call(qs=1028) == -5 and call(q=ctypes.c_void_p(264)) == -5
    need = lib.b200moe_paged_attn_fp8_workspace_bytes(2, 8, 2, 3)
    assert need > 0 and lib.b200moe_paged_attn_fp8_workspace_bytes(2, 8, 2, 1) == 0
    # Two, four and eight splits of few sequences merge without one.
    assert lib.b200moe_paged_attn_fp8_workspace_bytes(2, 8, 2, 8) == 0
    assert lib.b200moe_paged_attn_fp8_workspace_bytes(200, 8, 2, 8) > 0
    assert call(splits=3, ws=PTR, ws_bytes=need - 1) == -4 and call(splits=3) == -4
    assert call(batch=0) == 0


@pytest.mark.parametrize("batch,heads,longest", [(1, 1, 1), (1, 8, 700), (4, 1, 60001), (128, 8, 8192), (4000, 8, 10 ** 6), (1, 1, 2 ** 31 - 1)])
def test_split_counts_are_in_range(batch, heads, longest):
    for group in (1, 4, 16):
        assert 1 <= _lib.load().b200moe_paged_attn_fp8_num_splits(batch, heads * group, heads, longest) <= 64


def test_ops_refuse_cpu_tensors():
    i = torch.zeros(4, dtype=torch.int32)
    cache, scale = torch.zeros(2, 16, 2, 128).to(torch.float8_e4m3fn), torch.zeros(2, 2)
    x = torch.zeros(4, 2, 128, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA"):
        _C.paged_schedule(i, i, i.view(4, 1), i, i[:1], 16, i, torch.zeros(5, dtype=torch.int32), i, None, i[:1], i[:1])
    with pytest.raises(RuntimeError, match="CUDA"):
        _C.paged_store_kvcache_fp8(x, x, cache, cache, scale, scale, i)
    with pytest.raises(RuntimeError, match="CUDA"):
        _C.paged_attn_varlen_fp8(x, cache, cache, scale, scale, 0, i, i.view(4, 1), 0.1)


def test_oracle_codes_agree_with_torch():
    """The oracle's search over the code values against torch's conversion, on every bf16 value up to the
    largest code and on all ties between codes."""
    bits = torch.arange(-32768, 32768, dtype=torch.int32).to(torch.int16)
    x = bits.view(torch.bfloat16).float()
    x = x[x.abs() <= 448]
    want = x.to(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(decode_oracle.to_code_values(x.double().numpy()), want)
    codes = decode_oracle._CODES
    ties = torch.from_numpy((codes[1:] + codes[:-1]) / 2).float()
    assert np.array_equal(decode_oracle.to_code_values(ties.double().numpy()), ties.to(torch.float8_e4m3fn).double().numpy())
    assert decode_oracle.scale_ref(448.0) == 1.0 and decode_oracle.scale_ref(448.5) == 2.0 and decode_oracle.scale_ref(0.0) == 2.0 ** -32


def test_few_token_arguments():
    lib = _lib.load()

    def call(dtype=_lib.F32, tokens=4, experts=8, topk=2, hidden=256, inter=128, x=PTR, ws=PTR, ws_bytes=1 << 20):
        return lib.b200moe_few_tokens(x, PTR, dtype, PTR, PTR, PTR, tokens, experts, topk, hidden, inter, 1, ws, ws_bytes, None)

    assert lib.b200moe_few_tokens_max() == 32
    for bad in (dict(tokens=33), dict(tokens=-1), dict(experts=7), dict(topk=1), dict(hidden=250), dict(hidden=0), dict(inter=100),
                dict(inter=0), dict(hidden=(1 << 20) + 16), dict(inter=(1 << 20) + 8)):
        assert call(**bad) == -1, bad
    assert call(dtype=7) == -2 and call(x=None) == -3 and call(x=ctypes.c_void_p(264)) == -5
    need = lib.b200moe_few_tokens_workspace_bytes(4, 128)
    assert need == 4 * 2 * 128 * 4 and call(ws_bytes=need - 1) == -4 and call(ws=None) == -4
    assert call(tokens=0) == 0


def test_few_token_layer_arguments():
    from electrock_infer_b200.layers.moe import FusedMoE, fused_experts
    for bad in (dict(few_token_limit=33), dict(few_token_limit=-1)):
        with pytest.raises(ValueError):
            FusedMoE(8, 2, 64, 256, tp_size=1, **bad)
    with pytest.raises(ValueError):
        FusedMoE(4, 2, 64, 256, tp_size=1, few_token_limit=4)
    plain, few = FusedMoE(8, 2, 64, 256, tp_size=1), FusedMoE(8, 2, 64, 256, tp_size=1, few_token_limit=4)
    assert [plain.takes_few_tokens(n) for n in (0, 1, 32)] == [False] * 3
    assert [few.takes_few_tokens(n) for n in (0, 1, 4, 5)] == [False, True, True, False]
    with pytest.raises(RuntimeError, match="CUDA"):
        fused_experts(torch.zeros(4, 256, dtype=torch.bfloat16), torch.zeros(8, 512, 256, dtype=torch.bfloat16),
                      torch.zeros(8, 256, 256, dtype=torch.bfloat16), torch.zeros(4, 8), 2, few_tokens=True)
