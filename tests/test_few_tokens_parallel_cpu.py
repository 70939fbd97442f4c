"""``few_token_limit`` under tensor parallelism, over gloo with the oracle in place of the kernels."""
import os

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from electrock_infer_b200.layers.moe import FusedMoE
from electrock_infer_b200.layers.moe.mixtral_moe import MixtralMoE
from electrock_infer_b200.synthetic import MoEWorkload, make_inputs

WORLD = 2


def test_the_peer_exchange_is_refused_where_it_would_not_be_used():
    for cls in (FusedMoE, MixtralMoE):
        reduces = {"reduce_results": True} if cls is FusedMoE else {}
        with pytest.raises(ValueError, match="peer"):
            cls(8, 2, 64, 256, tp_size=2, tp_exchange="peer", few_token_limit=4, **reduces)
        cls(8, 2, 64, 256, tp_size=2, tp_exchange="peer", **reduces)
        cls(8, 2, 64, 256, tp_size=1, tp_exchange="peer", few_token_limit=4, **reduces)      # nothing to exchange
        for other in ("auto", "nccl"):
            cls(8, 2, 64, 256, tp_size=2, tp_exchange=other, few_token_limit=4, **reduces)
    FusedMoE(8, 2, 64, 256, tp_size=2, tp_exchange="peer", few_token_limit=4)                # no sum over ranks


def _worker(rank, result_dir):
    from electrock_infer_b200.layers.moe import mixtral_moe
    from oracle import moe_oracle
    dist.init_process_group("gloo", init_method=f"file://{result_dir}/rendezvous", rank=rank, world_size=WORLD)
    seen = []

    def cpu_fused_experts(hidden_states, w1, w2, gating_output, topk, renormalize, inplace, activation="silu",
                          gate_weight=None, tp_reduce=None, few_tokens=False):
        assert tp_reduce is None
        seen.append(few_tokens)
        if gate_weight is not None:
            gating_output = hidden_states @ gate_weight.t()
        hidden_states.copy_(moe_oracle.moe_block_ref(hidden_states, w1, w2, gating_output, topk, renormalize))
        return hidden_states

    mixtral_moe.fused_experts = cpu_fused_experts  # this process only
    wl = MoEWorkload("tp", 9, 32, 64, dtype=torch.float32, seed=19)
    full = make_inputs(wl)
    gate = torch.randn(8, 32, generator=torch.Generator().manual_seed(1))
    errs = []
    for block in (FusedMoE(8, 2, 32, 64, tp_size=WORLD, params_dtype=torch.float32, reduce_results=True, few_token_limit=8),
                  MixtralMoE(8, 2, 32, 64, tp_size=WORLD, params_dtype=torch.float32, few_token_limit=8)):
        layer = block if isinstance(block, FusedMoE) else block.experts
        for e in range(8):
            layer.weight_loader(layer.w13_weight, full["w13"][e, :64], "w1", e)
            layer.weight_loader(layer.w13_weight, full["w13"][e, 64:], "w3", e)
            layer.weight_loader(layer.w2_weight, full["w2"][e], "w2", e)
        if block is not layer:
            block.gate.weight.data.copy_(gate)
        for tokens in (1, 8, 9):
            x = full["x"][:tokens].clone()
            logits = full["logits"][:tokens] if block is layer else x @ gate.t()
            want = moe_oracle.moe_block_ref(x, full["w13"], full["w2"], logits)
            assert layer.peer_reduce_for(x) is None
            out = block(x, logits) if block is layer else block(x)
            errs.append((out - want).abs().max().item())
    torch.save({"errs": errs, "few": seen}, os.path.join(result_dir, f"few{rank}.pt"))
    dist.destroy_process_group()


def test_small_batches_are_summed_over_the_ranks(tmp_path):
    mp.spawn(_worker, args=(str(tmp_path),), nprocs=WORLD, join=True)
    for rank in range(WORLD):
        r = torch.load(tmp_path / f"few{rank}.pt")
        assert r["few"] == [True, True, False] * 2 and max(r["errs"]) < 1e-4, r
