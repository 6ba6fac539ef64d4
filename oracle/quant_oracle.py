"""Definitions in 64 bits of the 4-bit key-value cache and of the log
probabilities of tokens, in plain torch on the inputs' device.

A cache row (80 bytes) holds 128 values in four groups of 32: value d is
(code - 7.5) * scale + centre, its code nibble d % 8 of the 32-bit word
4 * (d % 32 // 8) + d // 32, centre and scale fp16 from byte 64 on.
"""
import numpy as np
import torch

DIM, GROUP, ROW = 128, 32, 80
LARGEST = 32768.0


def pack(x):
    """Rows [..., 128] of 16-bit values as cache rows, bit for bit what the definition's fp32 steps give (numpy)."""
    x = np.asarray(x.float().cpu().numpy(), np.float32).reshape(x.shape[:-1] + (4, GROUP))
    with np.errstate(all="ignore"):
        fine = (np.abs(x) <= np.float32(LARGEST)).all(-1)
        y = np.where(fine[..., None], x, np.float32(0))
        lo, hi = y.min(-1), y.max(-1)
        centre = ((lo + hi) * np.float32(0.5)).astype(np.float16)
        scale = ((hi - lo) / np.float32(15)).astype(np.float16)
        by = np.where(scale > 0, np.float32(1) / np.where(scale > 0, scale, 1).astype(np.float32), np.float32(0))
        u = (y - centre.astype(np.float32)[..., None]) * by[..., None].astype(np.float32) + np.float32(7.5)
    code = np.clip(np.rint(u), 0, 15).astype(np.uint32)
    code = np.where(fine[..., None], code, 8).astype(np.uint32).reshape(x.shape[:-2] + (4, 4, 8))   # group, eight, nibble
    word = np.zeros(code.shape[:-1], np.uint32)
    for n in range(8):
        word |= code[..., n] << np.uint32(4 * n)
    word = np.ascontiguousarray(np.swapaxes(word, -1, -2)).reshape(x.shape[:-2] + (16,))            # eight, group
    par = np.stack([centre, scale], -1).view(np.uint16)
    par = np.where(fine[..., None], par, np.uint16(0x7FFF)).astype(np.uint16).reshape(x.shape[:-2] + (8,))
    rows = np.concatenate([word.view(np.uint8), np.ascontiguousarray(par).view(np.uint8)], -1)
    return torch.from_numpy(rows)


def values(rows):
    """What cache rows [..., 80] stand for, [..., 128] in 64 bits."""
    d = torch.arange(DIM, device=rows.device)
    byte = rows[..., 16 * (d % 32 // 8) + 4 * (d // 32) + d % 8 // 2].int()
    code = (byte >> (4 * (d % 2)).int()) & 15
    par = rows[..., 64:].contiguous().view(torch.float16).double()
    return (code.double() - 7.5) * par[..., 2 * (d // 32) + 1] + par[..., 2 * (d // 32)]


def attend(query, key_cache, value_cache, table, q_lens, kv_lens, scale, causal):
    """Attention over the cache: (out, lse, near), 64 bits, [tokens, heads, 128] and [tokens, heads]. near: what the
    rounding bounds are relative to, as (sum of softmax * |value|, the largest scale * sum |query * key|). Pages
    outside the pool are zeros."""
    T, H, _ = query.shape
    blocks, page, kvh, _ = key_cache.shape
    dev = query.device
    out = torch.zeros((T, H, DIM), dtype=torch.float64, device=dev)
    lse = torch.full((T, H), float("-inf"), dtype=torch.float64, device=dev)
    size = torch.zeros((T, H, DIM), dtype=torch.float64, device=dev)
    reach = torch.zeros((T, H), dtype=torch.float64, device=dev)
    first = 0
    for b, (q, n) in enumerate(zip(list(q_lens), list(kv_lens))):
        q, n = int(q), min(int(n), table.shape[1] * page)
        if q == 0:
            continue
        mine = slice(first, first + q)
        first += q
        if n <= 0:
            continue
        ids = table[b, : (n + page - 1) // page].long()
        good = ((ids >= 0) & (ids < blocks))[:, None].expand(-1, page).reshape(-1)[:n]
        at = ids.clamp(0, blocks - 1)
        i, t = torch.arange(q, device=dev)[:, None], torch.arange(n, device=dev)
        hidden = (t > n - q + i) if causal else torch.zeros((q, n), dtype=torch.bool, device=dev)
        for h in range(kvh):
            k = torch.where(good[:, None], values(key_cache[at, :, h].reshape(-1, ROW)[:n]), 0.0)
            v = torch.where(good[:, None], values(value_cache[at, :, h].reshape(-1, ROW)[:n]), 0.0)
            for g in range(h * (H // kvh), (h + 1) * (H // kvh)):
                x = query[mine, g].double()
                s = (x @ k.T * scale).masked_fill(hidden, float("-inf"))
                top = s.amax(-1, keepdim=True)
                e = torch.exp(s - torch.where(torch.isinf(top), 0.0, top)).masked_fill(hidden, 0.0)
                total = e.sum(-1, keepdim=True)
                p = e / torch.where(total == 0, 1.0, total)
                w = torch.where(v.isfinite(), v, 0.0) if causal else v   # (hidden values are no part of any sum)
                out[mine, g], size[mine, g] = p @ w, p @ w.abs()
                lse[mine, g] = (torch.log(total) + top).squeeze(-1)
                reach[mine, g] = (x.abs() @ k.abs().nan_to_num(0.0).T).amax(-1) * scale
    return out, lse, (size, reach)


def logprobs(logits, tokens, top):
    """(logprob, entropy, rank, top_logprobs, top_tokens): 64 bits and whole numbers."""
    x = logits.double()
    N, V = x.shape
    top_x = x.amax(-1, keepdim=True)
    d = x - top_x
    e = torch.exp(d)
    total = e.sum(-1, keepdim=True)
    norm = torch.log(total)
    entropy = (norm - torch.where(e == 0, 0.0, e * d).sum(-1, keepdim=True) / total).squeeze(1)
    order = torch.where(x.isnan(), float("-inf"), x)
    place = torch.sort(order, dim=-1, descending=True, stable=True).indices
    rank = torch.empty_like(place)
    rank.scatter_(1, place, torch.arange(V, device=x.device).expand(N, V).contiguous())
    given = (tokens >= 0) & (tokens < V)
    at = tokens.clamp(0, V - 1)[:, None]
    mine = torch.where(given, (d.gather(1, at) - norm).squeeze(1), float("-inf"))
    return (mine, entropy, torch.where(given, rank.gather(1, at).squeeze(1), -1), d.gather(1, place[:, :top]) - norm,
            place[:, :top])
