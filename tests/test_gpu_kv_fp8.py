"""The 8-bit paged cache: the store against its definition in 64 bits (equal), attention against 64-bit
attention over the values that the codes stand for.

Bound of an attention output, with u = half a unit in the last place of its type:
  |err| <= u |want| + A (2^-11 + 2 d) + n 2^-25 max|v|,   A = sum_j p_j |v_j|
2^-11: P rounded to fp16 (normal numbers); n 2^-25 max|v|: probabilities below fp16's normal range, whose
rounding is absolute (the sum of probabilities is at least 1); d bounds the error of a score: 128
products accumulated in fp32, the tensor cores truncating, is at most 128 * 2^-23 of sum_d |q_d k_d| * scale,
and it enters both the numerator and the sum.
"""
import math

import numpy as np
import pytest
import torch

from electrock_infer_b200 import _C, _lib
from oracle import decode_oracle

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F8 = torch.float8_e4m3fn
HALF_ULP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def random_cache(blocks, block_size, heads, seed, spread=3):
    g = torch.Generator().manual_seed(seed)
    codes = (torch.randn(blocks, block_size, heads, 128, generator=g) * 100).clamp(-448, 448).to(F8)
    scale = torch.exp2(torch.randint(-7 - spread, -7 + spread + 1, (blocks, heads), generator=g).float())
    return codes, scale


# ---------------------------------------------------------------------------------------- store
def check_store(key, value, slots, blocks, block_size, seed=0, spread=3, k_scale=None, prepare=None):
    """Runs the store on random old contents and compares codes and scales with the definition."""
    heads = key.size(1)
    k_cache, ks = random_cache(blocks, block_size, heads, seed, spread)
    v_cache, vs = random_cache(blocks, block_size, heads, seed + 1, spread)
    if k_scale is not None:
        ks = k_scale
    d = [t.to(DEV) for t in (k_cache, v_cache, ks, vs)]
    dk, dv = (key.to(DEV), value.to(DEV)) if prepare is None else prepare(key, value)
    _C.paged_store_kvcache_fp8(dk, dv, *d, slots.to(DEV))
    torch.cuda.synchronize()
    for x, cache, scale, got_cache, got_scale in ((key, k_cache, ks, d[0], d[2]), (value, v_cache, vs, d[1], d[3])):
        want, want_scale = decode_oracle.paged_store_fp8_ref(x.double().numpy(), cache.double().numpy(),
                                                             scale.double().numpy(), slots.tolist())
        assert np.array_equal(got_scale.cpu().double().numpy(), want_scale, equal_nan=True)
        assert np.array_equal(got_cache.cpu().double().numpy(), want, equal_nan=True)


def request_slots(starts, news, block_size, blocks, seed):
    """Slot map of requests one after the other on pages dealt out at random."""
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(blocks, generator=g).tolist()
    slots, at = [], 0
    for a, n in zip(starts, news):
        pages = order[at: at - (-(a + n) // block_size)]
        at += len(pages)
        slots += [pages[p // block_size] * block_size + p % block_size for p in range(a, a + n)]
    assert at <= blocks
    return torch.tensor(slots, dtype=torch.int32)


def rows(n, heads, dtype, seed, loud=2.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, heads, 128, generator=g) * torch.exp2(torch.randn(n, 1, 1, generator=g) * loud)
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("heads,block_size,starts,news", [
    (8, 256, [0], [1]),
    (8, 256, [5, 255, 256, 511, 0], [1] * 5),                  # decode, page edges
    (1, 16, [0, 3, 15, 16], [40, 13, 1, 200]),
    (2, 48, [47, 0, 10], [1, 300, 38]),
    (3, 32, [1, 31, 7], [31, 33, 17]),                         # runs of 31, 32, 1, 17
    (4, 64, [0, 0, 0], [15, 16, 64]),
    (8, 256, [100, 0], [900, 513]),
    (2, 600, [100, 0], [700, 600]),                            # runs longer than one window
    (5, 1, [0, 2], [7, 5]),                                    # a page for every token
    (2, 16, list(range(60)), [1] * 60),
])
def test_store_equals_definition(heads, block_size, starts, news, dtype):
    blocks = sum(-(-(a + n) // block_size) for a, n in zip(starts, news)) + 2
    slots = request_slots(starts, news, block_size, blocks, seed=len(news))
    n = int(slots.numel())
    check_store(rows(n, heads, dtype, 1), rows(n, heads, dtype, 2), slots, blocks, block_size)


def test_store_of_many_tokens():
    starts, news = [0, 77, 1000], [4000, 500, 3]
    slots = request_slots(starts, news, 128, 60, seed=4)
    n = int(slots.numel())
    check_store(rows(n, 2, torch.bfloat16, 1), rows(n, 2, torch.bfloat16, 2), slots, 60, 128)


@pytest.mark.parametrize("gap", [1, 20, 300, 1500])
def test_store_with_skipped_tokens(gap):
    """Skipped entries before, between and behind the tokens of a page, more of them than any window."""
    real = request_slots([3, 0], [90, 200], 64, 9, seed=8).tolist()
    slots = [-1] * gap + real[:40] + [-1] * gap + real[40:41] + [10 ** 6, -7] + real[41:] + [2 ** 31 - 1] * gap
    slots = torch.tensor(slots, dtype=torch.int32)
    check_store(rows(len(slots), 2, torch.bfloat16, 1), rows(len(slots), 2, torch.bfloat16, 2), slots, 9, 64)


def test_store_with_nothing_to_do():
    slots = torch.full((700,), -1, dtype=torch.int32)
    check_store(rows(700, 2, torch.bfloat16, 1), rows(700, 2, torch.bfloat16, 2), slots, 3, 16)
    empty = torch.empty(0, 2, 128, dtype=torch.bfloat16)
    check_store(empty, empty, slots[:0], 3, 16)


def test_store_in_any_order_within_a_page():
    slots = torch.cat([torch.randperm(64) + 64 * p for p in (2, 0, 5)]).to(torch.int32)
    check_store(rows(192, 2, torch.float16, 1), rows(192, 2, torch.float16, 2), slots, 6, 64)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_store_of_strided_rows(dtype):
    n, heads = 37, 4
    slots = request_slots([9], [n], 16, 4, seed=2)

    def prepare(key, value):
        qkv = torch.zeros(n, 3 * heads * 128, dtype=dtype, device=DEV)
        k = qkv[:, heads * 128: 2 * heads * 128].view(n, heads, 128)
        v = qkv[:, 2 * heads * 128:].view(n, heads, 128)
        k.copy_(key)
        v.copy_(value)
        return k, v

    check_store(rows(n, heads, dtype, 1), rows(n, heads, dtype, 2), slots, 4, 16, prepare=prepare)


def test_store_of_extreme_values():
    """Largest codes, ties, subnormal codes, zeros, infinities, NaN, values beyond the scales' range."""
    x = torch.zeros(48, 1, 128, dtype=torch.float32)
    x[0, 0, :4] = torch.tensor([448.0, 449.0, 464.0, 480.0])
    x[1, 0, :6] = torch.tensor([1.0625, 1.1875, 2.0 ** -9, 2.0 ** -10, 1.5 * 2.0 ** -9, 2.0 ** -20])
    x[2, 0, 0], x[2, 0, 1] = math.inf, -math.inf
    x[3, 0, 0] = math.nan
    x[16, 0, 5] = 1e30                       # beyond the range: saturates
    x[17, 0, 5] = 2.0 ** -41                 # the smallest value there is a code for
    x[32:, 0, :] = 0.0                       # a page of zeros
    x[32, 0, 0] = -0.0
    slots = torch.arange(48, dtype=torch.int32)
    check_store(x, x.flip(2).contiguous(), slots, 4, 16)
    for sub in ([16], [32, 33], [3], [2]):   # alone, into pages with old contents or begun anew
        check_store(x[sub], x[sub], torch.arange(17, 17 + len(sub), dtype=torch.int32), 4, 16)
        check_store(x[sub], x[sub], torch.arange(16, 16 + len(sub), dtype=torch.int32), 4, 16)


@pytest.mark.parametrize("value", [0.0, -1.0, math.nan, math.inf, 1e-38])
def test_store_into_pages_with_unusable_scales(value):
    scale = torch.full((4, 2), value)
    check_store(rows(5, 2, torch.bfloat16, 1), rows(5, 2, torch.bfloat16, 2), torch.arange(20, 25, dtype=torch.int32), 4, 16,
                k_scale=scale)


def test_store_token_by_token_grows_the_scale():
    """A page filled by single tokens of growing size: every step against the definition."""
    k_cache, ks = random_cache(3, 32, 2, 7)
    v_cache, vs = random_cache(3, 32, 2, 8)
    d = [t.to(DEV) for t in (k_cache, v_cache, ks, vs)]
    want = [k_cache.double().numpy(), ks.double().numpy()]
    for i in range(32):
        x = (rows(1, 2, torch.bfloat16, 100 + i).float() * 1.6 ** i).to(torch.bfloat16)
        slot = torch.tensor([32 + i], dtype=torch.int32)
        _C.paged_store_kvcache_fp8(x.to(DEV), x.to(DEV), *d, slot.to(DEV))
        want = decode_oracle.paged_store_fp8_ref(x.double().numpy(), want[0], want[1], slot.tolist())
        assert np.array_equal(d[0].cpu().double().numpy(), want[0])
        assert np.array_equal(d[2].cpu().double().numpy(), want[1])


def test_store_refusals():
    k_cache, ks = (t.to(DEV) for t in random_cache(4, 16, 2, 1))
    v_cache, vs = (t.to(DEV) for t in random_cache(4, 16, 2, 2))
    x = rows(3, 2, torch.bfloat16, 1).to(DEV)
    slots = torch.arange(3, dtype=torch.int32, device=DEV)
    ok = dict(K=x, V=x, K_cache=k_cache, V_cache=v_cache, K_scale=ks, V_scale=vs, slot_mapping=slots)
    _C.paged_store_kvcache_fp8(**ok)
    odd = torch.zeros(3, 2 * 128 + 4, dtype=torch.bfloat16, device=DEV)[:, :256].view(3, 2, 128)
    for bad in (dict(K=x.cpu()), dict(K=x[:2]), dict(K=x.float()), dict(K=x.double(), V=x.double()), dict(K=odd, V=odd),
                dict(K=x.transpose(0, 1)), dict(K_cache=k_cache.view(torch.uint8)), dict(K_cache=k_cache[:3]),
                dict(K_scale=ks[:3]), dict(V_scale=vs.double()), dict(slot_mapping=slots.long()), dict(slot_mapping=slots[:2]),
                dict(K=x[..., :64].contiguous(), V=x[..., :64].contiguous()),
                dict(K_cache=k_cache.transpose(0, 1)), dict(K=x.view(-1)[1:1 + 256].view(1, 2, 128))):
        with pytest.raises(RuntimeError):
            _C.paged_store_kvcache_fp8(**{**ok, **bad})


# ------------------------------------------------------------------------------------ attention
def attn_case(lens, q_heads, kv_heads, block_size, dtype, seed, q_size=1.0):
    g = torch.Generator().manual_seed(seed)
    width = max(1, max(-(-n // block_size) for n in lens))
    blocks = len(lens) * width + 1
    k_cache, ks = random_cache(blocks, block_size, kv_heads, seed + 1)
    v_cache, vs = random_cache(blocks, block_size, kv_heads, seed + 2)
    table = torch.randperm(blocks, generator=g)[: len(lens) * width].view(len(lens), width).to(torch.int32)
    q = (torch.randn(len(lens), q_heads, 128, generator=g) * q_size).to(dtype)
    return {"q": q, "k_cache": k_cache, "v_cache": v_cache, "k_scale": ks, "v_scale": vs,
            "lens": torch.tensor(lens, dtype=torch.int32), "table": table, "scale": 128 ** -0.5}


def attend(c, splits=0, max_len=0, q=None, table=None):
    out = _C.paged_attn_varlen_fp8(c["q"].to(DEV) if q is None else q, c["k_cache"].to(DEV), c["v_cache"].to(DEV),
                                   c["k_scale"].to(DEV), c["v_scale"].to(DEV), max_len, c["lens"].to(DEV),
                                   c["table"].to(DEV) if table is None else table, c["scale"], num_splits=splits)
    torch.cuda.synchronize()
    return out.cpu()


def check_attn(c, got):
    want, mag, reach = decode_oracle.paged_attn_fp8_ref(c["q"], c["k_cache"], c["v_cache"], c["k_scale"], c["v_scale"],
                                                        c["lens"], c["table"], c["scale"])
    d = 128 * 2.0 ** -23 * reach.double()[:, None, None]
    vmax = float((c["v_cache"].float().abs().nan_to_num(0).amax((1, 3)) * c["v_scale"]).max())
    n = c["lens"].clamp(min=0).double()[:, None, None]
    bound = (HALF_ULP[c["q"].dtype] * want.abs() + mag * (2.0 ** -11 + 2 * d) + n * 2.0 ** -25 * vmax) * (1 + 2.0 ** -7)
    err = (got.double() - want).abs()
    assert torch.isfinite(got.float()).all()
    assert bool((err <= bound).all()), (err - bound).max().item()
    for b, length in enumerate(c["lens"].tolist()):
        if length <= 0:
            assert not got[b].any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("q_heads,kv_heads,block_size,lens,splits", [
    (32, 8, 256, [1, 15, 16, 17, 31, 32, 33, 255, 256, 257, 1000], 0),
    (32, 8, 256, [700], 0),
    (8, 8, 16, [33, 200, 1], 1),                               # no sharing
    (8, 1, 16, [129, 64, 640], 2),
    (12, 4, 48, [100, 47, 48, 49], 2),                         # groups of 3
    (12, 4, 48, [300, 47, 1, 0, 2000], 4),
    (10, 2, 32, [900, 1, 0, 64, 333], 8),
    (16, 1, 64, [2048, 1, 0, 777], 8),
    (14, 2, 32, [5, 95], 1),                                   # groups of 7
    (9, 1, 64, [130, 63], 3),                                  # groups of 9: two head tiles
    (16, 1, 64, [2048, 1], 7),
    (32, 2, 112, [300, 113, 111], 5),
    (16, 1, 16, [4000], 64),
    (4, 1, 16, [20, 100], 64),                                 # more splits than chunks
    (32, 8, 256, [0, 5, 0, -3], 1),                            # empty contexts
    (32, 8, 256, [0, 5, 0], 3),
])
def test_attention_against_64_bits(q_heads, kv_heads, block_size, lens, splits, dtype):
    c = attn_case(lens, q_heads, kv_heads, block_size, dtype, seed=q_heads + len(lens))
    check_attn(c, attend(c, splits))


@pytest.mark.parametrize("size", [1e-20, 1e-3, 30.0])
def test_attention_with_small_and_large_queries(size):
    c = attn_case([77, 500], 8, 2, 32, torch.bfloat16, seed=3, q_size=size)
    check_attn(c, attend(c))


@pytest.mark.parametrize("scale", [0.0, -0.1, 1.0])
def test_attention_with_other_softmax_scales(scale):
    c = {**attn_case([77, 500, 5], 8, 2, 32, torch.float16, seed=3), "scale": scale}
    for splits in (1, 3):
        check_attn(c, attend(c, splits))


def test_attention_where_scales_differ_by_page():
    """Pages whose scales lie up to 2^40 apart, the loud ones with vanishing weight."""
    c = attn_case([320, 47], 8, 2, 16, torch.bfloat16, seed=5)
    g = torch.Generator().manual_seed(1)
    c["v_scale"] = torch.exp2(torch.randint(-24, 17, c["v_scale"].shape, generator=g).float())
    c["k_scale"] = torch.exp2(torch.randint(-12, -5, c["k_scale"].shape, generator=g).float())
    check_attn(c, attend(c, 1))
    check_attn(c, attend(c, 4))


def test_attention_with_strided_queries_and_table():
    c = attn_case([40, 200, 3], 16, 4, 32, torch.float16, seed=6)
    fused = torch.zeros(3, 3, 16 * 128, dtype=torch.float16, device=DEV)
    q = fused[:, 1].view(3, 16, 128)
    q.copy_(c["q"])
    wide = torch.full((3, 20), 10 ** 6, dtype=torch.int32, device=DEV)
    table = wide[:, 2: 2 + c["table"].size(1)]
    table.copy_(c["table"])
    for splits in (1, 3):
        check_attn(c, attend(c, splits, q=q, table=table))


def test_attention_ignores_what_lies_behind_the_context():
    """NaN codes and NaN scales behind the context, and table entries that name no page."""
    c = attn_case([40, 1, 95], 8, 2, 32, torch.bfloat16, seed=9)
    want = attend(c, 1)
    for b, n in enumerate([40, 1, 95]):
        last = int(c["table"][b, n // 32])
        c["k_cache"][last, n % 32:] = math.nan
        c["v_cache"][last, n % 32:] = math.nan
        for j in range(-(-n // 32), c["table"].size(1)):
            c["k_scale"][c["table"][b, j]] = math.nan
            c["table"][b, j] = -1 if j % 2 else 10 ** 7
    for splits in (1, 2):
        got = attend(c, splits)
        check_attn({**c, "k_scale": c["k_scale"].nan_to_num(1.0)}, got)
    assert torch.equal(attend(c, 1), want)


def test_attention_passes_a_nan_of_the_context_on():
    c = attn_case([64, 64], 8, 2, 32, torch.bfloat16, seed=9)
    c["k_cache"][c["table"][0, 0], 5, 1, 3] = math.nan
    for splits in (1, 2):
        got = attend(c, splits).float()
        assert torch.isnan(got[0, 4:]).all() and torch.isfinite(got[0, :4]).all() and torch.isfinite(got[1]).all()


@pytest.mark.parametrize("max_len", [1, 100, 999, 10 ** 9])
@pytest.mark.parametrize("splits", [2, 5, 8, 37])
def test_attention_with_any_idea_of_the_longest_context(max_len, splits):
    """Contexts longer than max_seqlen_k are still attended to in full."""
    c = attn_case([999, 30, 0, 512], 8, 2, 16, torch.float16, seed=4)
    check_attn(c, attend(c, splits, max_len=max_len))


def test_attention_lengths_beyond_the_table_are_cut():
    c = attn_case([64, 60], 4, 1, 32, torch.bfloat16, seed=2)
    want = attend({**c, "lens": torch.tensor([64, 64], dtype=torch.int32)}, 1)
    assert torch.equal(attend({**c, "lens": torch.tensor([2 ** 31 - 1, 10 ** 6], dtype=torch.int32)}, 1), want)


def test_attention_at_offsets_past_32_bits():
    """A cache of more than 2^32 bytes: pages at its far end are stored to and read."""
    blocks, bs, heads = 135000, 16, 16     # 135000 * 16 * 16 * 128 B = 4.4e9
    k = torch.zeros(blocks, bs, heads, 128, dtype=torch.uint8, device=DEV).view(F8)
    v = torch.zeros(blocks, bs, heads, 128, dtype=torch.uint8, device=DEV).view(F8)
    ks, vs = torch.zeros(blocks, heads, device=DEV), torch.zeros(blocks, heads, device=DEV)
    pages = [blocks - 1, 3, blocks - 2]
    slots = torch.tensor([p * bs + i for p in pages for i in range(bs)][:45], dtype=torch.int32)
    key, value = rows(45, heads, torch.bfloat16, 1, 0.5), rows(45, heads, torch.bfloat16, 2, 0.5)
    _C.paged_store_kvcache_fp8(key.to(DEV), value.to(DEV), k, v, ks, vs, slots.to(DEV))
    q = torch.randn(1, 32, 128).to(torch.bfloat16)
    got = _C.paged_attn_varlen_fp8(q.to(DEV), k, v, ks, vs, 45, torch.tensor([45], dtype=torch.int32, device=DEV),
                                   torch.tensor([pages], dtype=torch.int32, device=DEV), 128 ** -0.5)
    small = {"q": q, "k_cache": k[pages].cpu(), "v_cache": v[pages].cpu(), "k_scale": ks[pages].cpu(),
             "v_scale": vs[pages].cpu(), "lens": torch.tensor([45], dtype=torch.int32),
             "table": torch.tensor([[0, 1, 2]], dtype=torch.int32), "scale": 128 ** -0.5}
    check_attn(small, got.cpu())
    want, _ = decode_oracle.paged_store_fp8_ref(key.double().numpy(), np.zeros((3, bs, heads, 128)), np.zeros((3, heads)), range(45))
    assert np.array_equal(small["k_cache"].double().numpy(), want)


def test_attention_is_the_same_every_time_and_on_other_streams():
    c = attn_case([700, 90, 2000], 32, 8, 64, torch.bfloat16, seed=12)
    d = {k: (t.to(DEV) if torch.is_tensor(t) else t) for k, t in c.items()}
    call = lambda: _C.paged_attn_varlen_fp8(d["q"], d["k_cache"], d["v_cache"], d["k_scale"], d["v_scale"], 2000,  # noqa: E731
                                            d["lens"], d["table"], d["scale"], num_splits=5)
    first = call()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(call())
    torch.cuda.synchronize()
    assert all(torch.equal(o, first) for o in outs)


def test_captured_attention_replayed_at_the_same_time():
    """Two graphs with splits that go through a workspace, replayed on two streams at once: none shares scratch."""
    c = attn_case([700, 90, 2000], 32, 8, 64, torch.bfloat16, seed=12)
    d = {k: (t.to(DEV) if torch.is_tensor(t) else t) for k, t in c.items()}
    qs = [d["q"], (d["q"].float() * -0.5).to(torch.bfloat16)]
    call = lambda q: _C.paged_attn_varlen_fp8(q, d["k_cache"], d["v_cache"], d["k_scale"], d["v_scale"], 2000, d["lens"],  # noqa: E731
                                              d["table"], d["scale"], num_splits=7)
    want = [call(q) for q in qs]
    graphs, outs = [], []
    for q in qs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(q))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    for _ in range(30):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, want))


def test_attention_refusals():
    c = attn_case([10, 20], 32, 8, 32, torch.bfloat16, seed=1)
    d = {k: (v.to(DEV) if torch.is_tensor(v) else v) for k, v in c.items()}
    ok = dict(Q=d["q"], K_cache=d["k_cache"], V_cache=d["v_cache"], K_scale=d["k_scale"], V_scale=d["v_scale"],
              max_seqlen_k=0, context_lens=d["lens"], block_table=d["table"], softmax_scale=0.1)
    _C.paged_attn_varlen_fp8(**ok)
    small = torch.zeros(5, 8, 8, 128, dtype=torch.uint8, device=DEV).view(F8)
    for bad in (dict(Q=d["q"].float()), dict(Q=d["q"][..., :64].contiguous()), dict(Q=d["q"][:, :30].contiguous()),
                dict(Q=d["q"].cpu()), dict(Q=torch.zeros(2, 8 * 17, 128, dtype=torch.bfloat16, device=DEV)),
                dict(K_cache=d["k_cache"].view(torch.uint8)), dict(V_cache=d["v_cache"][:1]), dict(K_scale=d["k_scale"][:, :4]),
                dict(context_lens=d["lens"].long()), dict(context_lens=d["lens"][:1]), dict(block_table=d["table"].long()),
                dict(block_table=d["table"][:1]), dict(block_table=torch.zeros(2, 4, dtype=torch.int32, device=DEV)[:, ::2]),
                dict(num_splits=65), dict(K_cache=small, V_cache=small, K_scale=torch.ones(5, 8, device=DEV), V_scale=torch.ones(5, 8, device=DEV))):
        with pytest.raises(RuntimeError):
            _C.paged_attn_varlen_fp8(**{**ok, **bad})
    rc = _lib.load().b200moe_paged_attn_varlen_fp8(
        d["q"].data_ptr(), d["k_cache"].data_ptr(), d["v_cache"].data_ptr(), d["k_scale"].data_ptr(), d["v_scale"].data_ptr(),
        d["q"].data_ptr(), d["table"].data_ptr(), d["lens"].data_ptr(), _lib.BF16, 2, 32, 8, 128, 32 * 128, d["k_cache"].size(0),
        32, 1, 1, 0.1, 5, None, 0, torch.cuda.current_stream().cuda_stream)
    assert rc == -4  # no workspace for num_splits = 5
