"""CPU oracle of the decode-step operators: step tables, 8-bit paged cache, few-token expert layer.
TEST INFRASTRUCTURE ONLY.

Plain restatements of the definitions in include/b200moe.h, request by request and page by page, in
64-bit arithmetic.  Nothing in the product package imports this module.
"""
from __future__ import annotations

import math

import numpy as np
import torch

CODE_MAX = 448.0
INT_MAX = 2 ** 31 - 1


# ------------------------------------------------------------------------------------ step tables
def paged_schedule_ref(context_lens, new_lens, block_table, free_blocks, free_count, block_size,
                       num_rows):
    """One request after the other, with a Python list as the stack.  Returns a dict of numpy arrays;
    the inputs are not modified."""
    table = np.array(block_table, dtype=np.int64)
    requests, width = table.shape
    stack_mem = np.array(free_blocks, dtype=np.int64)
    top = min(max(int(free_count), 0), len(stack_mem))
    ctx = [min(max(int(c), 0), width * block_size) for c in context_lens]
    new = [int(n) for n in new_lens]
    # Pages of ended requests first.
    for i in range(requests):
        if new[i] < 0:
            for j in range(-(-ctx[i] // block_size)):
                if top < len(stack_mem):
                    stack_mem[top] = table[i, j]
                    top += 1
    avail = top
    seq = np.zeros(requests, np.int64)
    cu = np.zeros(requests + 1, np.int64)
    slots = np.full(num_rows, -1, np.int64)
    positions = np.zeros(num_rows, np.int64)
    refused, wanted, row = 0, 0, 0
    for i in range(requests):
        rows = max(new[i], 0)
        have = -(-ctx[i] // block_size)
        want = -(-(ctx[i] + rows) // block_size)
        fits = want <= width and row + rows <= num_rows
        need = want - have if rows and fits else 0
        wanted += need
        served = rows > 0 and fits and (need == 0 or wanted <= avail)
        if served:
            for j in range(have, want):
                top -= 1
                table[i, j] = stack_mem[top]
        elif rows:
            refused += 1
        for k in range(rows):
            if row + k >= num_rows:
                break
            pos = ctx[i] + k
            positions[row + k] = pos
            if served:
                page = table[i, pos // block_size]
                slot = page * block_size + pos % block_size
                if page >= 0 and slot <= INT_MAX:
                    slots[row + k] = slot
        row += rows
        seq[i] = 0 if new[i] < 0 else ctx[i] + (rows if served else 0)
        cu[i + 1] = min(row, num_rows)
    return {"block_table": table, "free_blocks": stack_mem, "seq_lens": seq, "cu_seqlens": cu,
            "slot_mapping": slots, "positions": positions, "free_count_out": top,
            "num_refused": refused}


# ------------------------------------------------------------------------------------ 8-bit cache
def _code_values() -> np.ndarray:
    """The 127 non-negative finite e4m3 values, by code."""
    vals = []
    for code in range(127):
        exp, man = code >> 3, code & 7
        vals.append((man / 8) * 2.0 ** -6 if exp == 0 else (1 + man / 8) * 2.0 ** (exp - 7))
    return np.array(vals)


_CODES = _code_values()


def to_code_values(x: np.ndarray) -> np.ndarray:
    """The e4m3 value nearest to every x; ties to the even code, saturating, NaN kept."""
    size = np.minimum(np.abs(x), CODE_MAX)
    hi = np.clip(np.searchsorted(_CODES, np.nan_to_num(size), side="left"), 0, 126)
    lo = np.maximum(hi - 1, 0)
    up, down = _CODES[hi] - size, size - _CODES[lo]
    pick = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    return np.where(np.isnan(x), np.nan, np.sign(x) * _CODES[pick])


def scale_ref(amax: float) -> float:
    """Smallest power of two in [2^-32, 2^32] with amax <= 448 * scale."""
    e = -32
    while e < 32 and amax > CODE_MAX * 2.0 ** e:
        e += 1
    return 2.0 ** e


def paged_store_fp8_ref(x, cache, scale, slots):
    """``x [tokens, heads, 128]``, ``cache [blocks, block_size, heads, 128]`` code values and
    ``scale [blocks, heads]`` as float64 arrays.  Returns the new (cache, scale)."""
    cache, scale = np.array(cache, dtype=np.float64), np.array(scale, dtype=np.float64)
    blocks, block_size, heads, _ = cache.shape
    pages: dict = {}
    for token, slot in enumerate(slots):
        if 0 <= slot < blocks * block_size:
            pages.setdefault(int(slot) // block_size, []).append((token, int(slot) % block_size))
    for page, items in pages.items():
        fresh = any(off == 0 for _, off in items)
        for h in range(heads):
            rows = np.stack([x[t, h] for t, _ in items])
            finite = np.abs(rows[np.isfinite(rows)])
            unit = scale_ref(float(finite.max()) if finite.size else 0.0)
            if not fresh:
                old = scale[page, h]
                old = 2.0 ** -32 if not old >= 2.0 ** -32 else min(old, 2.0 ** 32)
                if unit > old:
                    cache[page, :, h] = to_code_values(cache[page, :, h] * (old / unit))
                unit = max(unit, old)
            scale[page, h] = unit
            for (t, off), row in zip(items, rows):
                cache[page, off, h] = to_code_values(row / unit)
    return cache, scale


def paged_attn_fp8_ref(q, k_cache, v_cache, k_scale, v_scale, context_lens, block_table, softmax_scale):
    """float64 attention; also returns, per output, sum_j p_j |v_j| and the sequence's largest
    sum_d |q_d k_d| * softmax_scale, which error bounds are made of."""
    q = q.double()
    batch, q_heads, dim = q.shape
    block_size, kv_heads = k_cache.size(1), k_cache.size(2)
    group = q_heads // kv_heads
    out, mag = torch.zeros_like(q), torch.zeros_like(q)
    reach = torch.zeros(batch)
    for b, n in enumerate(context_lens.tolist()):
        if n <= 0:
            continue
        pages = block_table[b, : -(-n // block_size)].long()
        k = (k_cache[pages].double() * k_scale[pages].double()[:, None, :, None]).flatten(0, 1)[:n]
        v = (v_cache[pages].double() * v_scale[pages].double()[:, None, :, None]).flatten(0, 1)[:n]
        for h in range(q_heads):
            kh, vh = k[:, h // group], v[:, h // group]
            s = kh @ q[b, h] * softmax_scale
            p = torch.softmax(s, 0)
            out[b, h] = p @ vh
            mag[b, h] = p @ vh.abs()
            reach[b] = max(float(reach[b]), float((kh.abs() @ q[b, h].abs()).max() * abs(softmax_scale)))
    return out, mag, reach


# ------------------------------------------------------------------------------- few-token layer
def few_tokens_ref(x, logits, w13, w2, renormalize=True):
    """float64 top-2 layer; also returns sum over the addends of |w act w2| per output element."""
    x, w13, w2 = x.double(), w13.double(), w2.double()
    inter = w2.size(2)
    out, mag = torch.zeros_like(x), torch.zeros_like(x)
    for t in range(x.size(0)):
        row = logits[t].double().tolist()
        order = sorted(range(len(row)), key=lambda e: (-row[e], e))[:2]
        ex = [math.exp(v - max(row)) for v in row]
        probs = [ex[e] / sum(ex) for e in order]
        if renormalize:
            probs = [p / sum(probs) for p in probs]
        for e, w in zip(order, probs):
            z = w13[e] @ x[t]
            act = z[:inter] / (1 + torch.exp(-z[:inter])) * z[inter:] * w
            out[t] += w2[e] @ act
            mag[t] += w2[e].abs() @ act.abs()
    return out, mag
