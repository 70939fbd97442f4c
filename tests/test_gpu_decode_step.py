"""The decode-step operators in the order a server runs them: step tables, store, attention and expert layer
over a few dozen steps, eagerly and as one captured graph, against the definitions in 64 bits."""
import numpy as np
import pytest
import torch

from electrock_infer_b200 import _C
from electrock_infer_b200.layers.moe import FusedMoE
from oracle import decode_oracle
from test_gpu_kv_fp8 import HALF_ULP

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
R, HIDDEN, Q_HEADS, KV_HEADS, INTER, PAGE, WIDTH, POOL = 7, 512, 4, 2, 256, 16, 8, 40


class Model:
    """One layer without norms: projections by torch, everything else by the operators under test."""

    def __init__(self, rows, seed=0):
        g = torch.Generator().manual_seed(seed)
        rand = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
        self.rows = rows
        self.wqkv = (rand(HIDDEN, (Q_HEADS + 2 * KV_HEADS) * 128) * HIDDEN ** -0.5).to(DEV, torch.bfloat16)
        self.wo = (rand(Q_HEADS * 128, HIDDEN) * HIDDEN ** -0.5).to(DEV, torch.bfloat16)
        self.gate = rand(HIDDEN, 8).mul(HIDDEN ** -0.5 * 2).to(DEV, torch.bfloat16)
        self.moe = FusedMoE(8, 2, HIDDEN, INTER, params_dtype=torch.bfloat16, few_token_limit=32).to(DEV)
        self.moe.w13_weight.data.copy_((rand(8, 2 * INTER, HIDDEN) * HIDDEN ** -0.5).to(torch.bfloat16))
        self.moe.w2_weight.data.copy_((rand(8, HIDDEN, INTER) * INTER ** -0.5).to(torch.bfloat16))
        i32 = dict(dtype=torch.int32, device=DEV)
        self.lens, self.new, self.cu = torch.zeros(R, **i32), torch.zeros(R, **i32), torch.zeros(R + 1, **i32)
        self.table = torch.full((R, WIDTH), -1, **i32)
        self.free, self.count, self.refused = torch.arange(POOL, **i32), torch.tensor([POOL], **i32), torch.zeros(1, **i32)
        self.caches = [torch.zeros(POOL, PAGE, KV_HEADS, 128, device=DEV).to(torch.float8_e4m3fn) for _ in range(2)]
        self.scales = [torch.zeros(POOL, KV_HEADS, device=DEV) for _ in range(2)]

    def step(self, x, slots, positions):
        """One pass over the rows ``x``; returns what the checks need."""
        _C.paged_schedule(self.lens, self.new, self.table, self.free, self.count, PAGE, self.lens, self.cu, slots, positions,
                          self.count, self.refused)
        qkv = (x @ self.wqkv).view(x.size(0), Q_HEADS + 2 * KV_HEADS, 128)
        k, v = qkv[:, Q_HEADS:Q_HEADS + KV_HEADS], qkv[:, Q_HEADS + KV_HEADS:]
        _C.paged_store_kvcache_fp8(k, v, *self.caches, *self.scales, slots)
        last = (self.cu[1:].long() - 1).clamp(min=0)                     # the last row of each request
        q = qkv[last, :Q_HEADS]
        attn = _C.paged_attn_varlen_fp8(q, *self.caches, *self.scales, 0, self.lens, self.table, 128 ** -0.5)
        h = attn.view(R, -1) @ self.wo
        logits = (h @ self.gate).float()
        return {"k": k, "v": v, "q": q, "attn": attn, "h": h, "logits": logits, "out": self.moe(h.clone(), logits)}


class Shadow:
    """The same state kept by the definitions, on the CPU."""

    def __init__(self):
        self.lens, self.table = [0] * R, np.full((R, WIDTH), -1)
        self.free, self.count = np.arange(POOL), POOL
        self.cache = [np.zeros((POOL, PAGE, KV_HEADS, 128)) for _ in range(2)]
        self.scale = [np.zeros((POOL, KV_HEADS)) for _ in range(2)]

    def check(self, model, new, slots, got):
        want = decode_oracle.paged_schedule_ref(self.lens, new, self.table, self.free, self.count, PAGE, slots.numel())
        self.lens, self.table, self.free, self.count = (want["seq_lens"], want["block_table"], want["free_blocks"],
                                                        want["free_count_out"])
        assert np.array_equal(slots.cpu().numpy(), want["slot_mapping"])
        assert np.array_equal(model.lens.cpu().numpy(), self.lens) and int(model.count) == self.count
        for i, key in enumerate("kv"):
            self.cache[i], self.scale[i] = decode_oracle.paged_store_fp8_ref(
                got[key].cpu().double().numpy(), self.cache[i], self.scale[i], want["slot_mapping"])
            assert np.array_equal(model.scales[i].cpu().double().numpy(), self.scale[i])
            assert np.array_equal(model.caches[i].cpu().double().numpy(), self.cache[i])
        t = torch.from_numpy
        ref, mag, reach = decode_oracle.paged_attn_fp8_ref(
            got["q"].cpu(), t(self.cache[0]), t(self.cache[1]), t(self.scale[0]), t(self.scale[1]),
            torch.as_tensor(self.lens), t(self.table), 128 ** -0.5)
        vmax = float((np.abs(self.cache[1]).max((1, 3)) * self.scale[1]).max())
        bound = (HALF_ULP[torch.bfloat16] * ref.abs() + mag * (2.0 ** -11 + 2 ** -15 * reach.double()[:, None, None])
                 + 2.0 ** -25 * vmax * PAGE * WIDTH) * (1 + 2.0 ** -7)
        assert bool(((got["attn"].cpu().double() - ref).abs() <= bound).all())
        moe, _ = decode_oracle.few_tokens_ref(got["h"].cpu(), got["logits"].cpu(), model.moe.w13_weight.cpu(), model.moe.w2_weight.cpu())
        assert (got["out"].cpu().double() - moe).norm() <= 2.0 ** -8 * moe.norm() + 1e-30


def test_prompts_then_decoding_with_a_captured_graph():
    model, shadow = Model(rows=R), Shadow()
    g = torch.Generator(device=DEV).manual_seed(1)

    # Prompts of ragged length, some rows of padding.
    new = [20, 1, 33, 16, 7, 0, 48]
    rows = sum(new) + 3
    slots = torch.empty(rows, dtype=torch.int32, device=DEV)
    positions = torch.empty(rows, dtype=torch.int64, device=DEV)
    model.new.copy_(torch.tensor(new, dtype=torch.int32))
    x = torch.randn(rows, HIDDEN, generator=g, device=DEV).to(torch.bfloat16)
    shadow.check(model, new, slots, model.step(x, slots, positions))

    # Decode steps: one eagerly, then the same as a graph, replayed with other inputs; requests end, wait,
    # begin and are refused meanwhile.
    slots = torch.empty(R, dtype=torch.int32, device=DEV)
    positions = torch.empty(R, dtype=torch.int64, device=DEV)
    x = torch.empty(R, HIDDEN, dtype=torch.bfloat16, device=DEV)

    def inputs(lens):
        model.new.copy_(torch.tensor(lens, dtype=torch.int32))
        x.copy_(torch.randn(R, HIDDEN, generator=g, device=DEV))

    inputs([1] * R)
    shadow.check(model, [1] * R, slots, model.step(x, slots, positions))
    graph = torch.cuda.CUDAGraph()
    before = [t.clone() for t in (model.lens, model.table, model.free, model.count)]
    with torch.cuda.graph(graph):
        got = model.step(x, slots, positions)
    for now, old in zip((model.lens, model.table, model.free, model.count), before):
        assert torch.equal(now, old)          # capturing runs nothing
    plans = [[1] * R, [1, -1, 1, 1, -1, 1, 1], [1, 1, 0, 1, 1, 0, 1], [0, 1, -1, 0, 1, 1, -1]] + [[1] * R] * 6
    for plan in plans:
        inputs(plan)
        graph.replay()
        torch.cuda.synchronize()
        shadow.check(model, plan, slots, got)
    # Run every request into the end of its table row: refused ones keep their length.
    for _ in range(3):
        model.new.copy_(torch.tensor([40] + [0] * (R - 1), dtype=torch.int32))
        many = torch.randn(40, HIDDEN, generator=g, device=DEV).to(torch.bfloat16)
        more_slots = torch.empty(40, dtype=torch.int32, device=DEV)
        shadow.check(model, [40] + [0] * (R - 1), more_slots, model.step(many, more_slots, torch.empty(40, dtype=torch.int64, device=DEV)))
    assert int(model.refused) == 1
    inputs([1] * R)
    graph.replay()
    torch.cuda.synchronize()
    shadow.check(model, [1] * R, slots, got)
