"""The paged operators in plain 64-bit arithmetic, request by request."""
import numpy as np
import torch

GROUP = 32
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def ceil_div(a, b):
    return -(-a // b)


def plan(cached, fresh, table, stack, count, page, capacity):
    """One step with lists: the ended requests push, the others pop."""
    table, stack = table.copy(), stack.copy()
    held = list(stack[:count])
    for b, (c, f) in enumerate(zip(cached, fresh)):
        if f < 0:
            held += list(table[b, :ceil_div(c, page)])
    first_held = list(held)
    lengths, waiting, wanted = [], False, 0
    slots, positions = np.full(capacity, -1, np.int64), np.zeros(capacity, np.int32)
    query_begin = [0]
    for b, (c, f) in enumerate(zip(cached, fresh)):
        n = max(f, 0)
        have = ceil_div(c, page)
        need = 0 if f < 0 else ceil_div(c + n, page) - have
        wanted += need
        got = f >= 0 and (need == 0 or (not waiting and need <= len(held)))
        if f >= 0 and not got:
            waiting = True
        if got:
            for i in range(need):
                table[b, have + i] = held.pop()
        lengths.append(0 if f < 0 else c + n if got else c)
        for i in range(n):
            row, p = query_begin[-1] + i, c + i
            positions[row] = p
            if got:
                slots[row] = int(table[b, p // page]) * page + p % page
        query_begin.append(query_begin[-1] + n)
    for i in range(count, len(held)):
        stack[i] = held[i]
    return dict(table=table, free_pages=stack, free_left=len(held), lengths=lengths, query_begin=query_begin,
                key_begin=[0] + list(np.cumsum(lengths)), slots=slots, positions=positions, shortage=max(0, wanted - len(first_held)))


def quantized(x):
    """(quants 0..15, scales) of the groups of rows x, in float64; a NaN counts as 0."""
    g = torch.nan_to_num(x.double(), nan=0.0, posinf=np.inf, neginf=-np.inf).reshape(-1, GROUP)
    first = g.abs().argmax(1, keepdim=True)
    top = g.abs().amax(1, keepdim=True)
    first = (g.abs() == top).int().argmax(1, keepdim=True)
    d = (g.gather(1, first) / -8).clamp(-65504, 65504).half().double()
    q = ((g / torch.where(d == 0, torch.ones_like(d), d)) + 8.5).floor().clamp(0, 15)
    return torch.where(d == 0, torch.full_like(q, 8), q), d


def kept(x):
    q, d = quantized(x)
    return ((q - 8) * d).reshape(x.shape)


def attention(q, k, v, scale, causal=True):
    """q {n, heads, dim}, k / v {L, kv heads, dim} -> (result, sum of |weight value|, weights' total) in float64."""
    n, heads, _ = q.shape
    length, kv = k.shape[:2]
    group = heads // kv
    k, v = k.double().repeat_interleave(group, 1), v.double().repeat_interleave(group, 1)
    s = torch.einsum("nhd,lhd->hnl", q.double(), k) * scale
    if causal:
        i, j = torch.arange(n, device=q.device)[:, None], torch.arange(length, device=q.device)[None]
        s = s.masked_fill(j > length - n + i, -np.inf)
    if length == 0:
        z = torch.zeros(n, heads, v.shape[-1], dtype=torch.float64, device=q.device)
        return z, z, torch.ones(n, heads, 1, dtype=torch.float64, device=q.device)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -np.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    out = torch.einsum("hnl,lhd->nhd", p, torch.where(torch.isfinite(v), v, torch.zeros_like(v)))
    size = torch.einsum("hnl,lhd->nhd", p, torch.where(torch.isfinite(v), v.abs(), torch.zeros_like(v)))
    return out, size, total.permute(1, 0, 2)
