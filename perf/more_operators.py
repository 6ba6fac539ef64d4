"""The operators of a key-value cache held in 4 bits, and the log probabilities of
tokens, as measured work: keys and values quantised as they are written, read
back, attended to by single tokens, drafted tokens and chunks of prompts; the
log probability, entropy, rank and best alternatives of given tokens.

``listed()`` names the cases, ``draw()`` gives more of the same ranges,
``prepare()`` makes a case's inputs on the GPU and ``run()`` does one pass:
plain torch operations in 32 bits while ``own`` is false, this repository's
kernels while it is true. ``exact()`` is the definition in 64 bits and ``work()``
the bytes and operations that a pass cannot do without.
"""
import os
import sys

import torch

own = False

DIM = 128                     # values of a key or a value
GROUP = 32                    # values that share a centre and a scale
ROW = DIM // 2 + DIM // GROUP * 4  # bytes of a cache row: codes, then (centre, scale) per group in fp16
SCALE = DIM ** -0.5
GOLDEN = 0.6180339887498949
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # one user's chat, every head on this GPU: nothing but latency
        {"name": "attend, one request", "op": "attend", "batch": 1, "kv_heads": 8, "group": 4, "q_len": 1, "kv_lo": 900,
         "kv_hi": 900, "page": 16, "dtype": "bf16"},
        # a batch of mixed chats on small pages
        {"name": "attend, mixed batch", "op": "attend", "batch": 48, "kv_heads": 8, "group": 4, "q_len": 1, "kv_lo": 1,
         "kv_hi": 6001, "page": 16, "dtype": "bf16"},
        # a full batch of long chats
        {"name": "attend, full batch", "op": "attend", "batch": 128, "kv_heads": 8, "group": 8, "q_len": 1, "kv_lo": 1500,
         "kv_hi": 8200, "page": 64, "dtype": "bf16"},
        # a few very long documents, one key-value head of eight on this GPU
        {"name": "attend, long documents", "op": "attend", "batch": 3, "kv_heads": 1, "group": 8, "q_len": 1, "kv_lo": 60000,
         "kv_hi": 100000, "page": 128, "dtype": "bf16"},
        # the target model's pass over three drafted tokens and the one before them
        {"name": "attend, drafted tokens", "op": "attend", "batch": 24, "kv_heads": 8, "group": 5, "q_len": 4, "kv_lo": 4,
         "kv_hi": 5003, "page": 32, "dtype": "fp16"},
        # chunks of two prompts behind their context
        {"name": "attend, prompt chunk", "op": "attend", "batch": 2, "kv_heads": 8, "group": 4, "q_len": 512, "kv_lo": 4100,
         "kv_hi": 4601, "page": 64, "dtype": "fp16"},
        # the tokens of one decode step enter the cache
        {"name": "store, decode step", "op": "store", "tokens": 64, "kv_heads": 8, "page": 16, "dtype": "bf16"},
        # a batch of prompts enters the cache and is read back
        {"name": "store, prompts", "op": "store", "tokens": 20001, "kv_heads": 8, "page": 64, "dtype": "fp16"},
        # a cached context in 16 bits, for a prompt's own attention
        {"name": "read, context", "op": "read", "tokens": 60001, "kv_heads": 4, "page": 32, "dtype": "bf16"},
        # a few requests that ask for log probabilities
        {"name": "logprobs, small", "op": "logprobs", "rows": 4, "vocab": 32000, "top": 5, "dtype": "fp32"},
        # a full batch over a large vocabulary
        {"name": "logprobs, batch", "op": "logprobs", "rows": 128, "vocab": 128256, "top": 20, "dtype": "bf16"},
        # every token of a prompt is scored
        {"name": "logprobs, prompt", "op": "logprobs", "rows": 1500, "vocab": 128256, "top": 1, "dtype": "bf16"},
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(lo * (hi / lo) ** rng.random()))

    op = rng.choice(["attend", "attend", "attend", "store", "read", "logprobs", "logprobs"])
    two = rng.choice(["bf16", "fp16"])
    if op == "attend":
        batch, kvh, group = log(1, 128), rng.choice([1, 2, 4, 8, 8]), rng.choice([1, 2, 4, 5, 7, 8])
        q_len = rng.choice([1, 1, 1, 2, 3, 5, log(8, 512)])
        hi = log(1, 40000)
        hi = max(1, min(hi, 8000000 // (batch * kvh), 140000000 // (batch * kvh * group * q_len)))
        return {"op": op, "batch": batch, "kv_heads": kvh, "group": group, "q_len": q_len, "kv_lo": rng.randint(0, hi),
                "kv_hi": hi, "page": rng.choice([16, 32, 64, 128]), "dtype": two}
    if op == "logprobs":
        vocab = log(1000, 128256)
        return {"op": op, "rows": max(1, min(log(1, 2000), 190000000 // vocab)), "vocab": vocab,
                "top": rng.choice([0, 1, 5, 20, rng.randint(1, 32)]), "dtype": rng.choice(["fp32", "bf16", "bf16", "fp16"])}
    kvh = rng.choice([1, 2, 4, 8])
    return {"op": op, "tokens": min(log(1, 60000), 240000 // kvh), "kv_heads": kvh, "page": rng.choice([16, 32, 64, 128]),
            "dtype": two}


def _spread(n, lo, hi):
    """n whole numbers over [lo, hi], the same for every seed (work() counts them)."""
    return [lo + int((hi - lo + 1) * ((i * GOLDEN + 0.5) % 1.0)) for i in range(n)]


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * scale).to(dtype)


def _pages(lens, page):
    return sum((n + page - 1) // page for n in lens)


def prepare(case, seed):
    if own:
        here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vllm-hust-cascade-kernel_b200")
        if here not in sys.path:
            sys.path.insert(0, here)
        import cascade_kernel  # noqa: F401  registers torch.ops.npu.*
    g, op, dtype = _generator(seed), case["op"], DTYPES[case["dtype"]]
    s = {"op": op, "dtype": dtype}
    if op == "logprobs":
        N, V = case["rows"], case["vocab"]
        s["logits"] = _normal(g, (N, V), dtype, 2.5)
        # a sampled token is a likely one; one in eight of a prompt's is not
        pick = torch.rand((N, V), generator=g, device="cuda").clamp_(min=1e-30).log_().neg_().log_().neg_()
        sampled = torch.argmax(pick.add_(s["logits"]), -1)
        other = torch.randint(0, V, (N,), generator=g, device="cuda")
        s["tokens"] = torch.where(torch.randint(0, 8, (N,), generator=g, device="cuda") == 0, other, sampled)
        s["top"] = case["top"]
        return s
    page, kvh = case["page"], case["kv_heads"]
    lens = _spread(case["batch"], case["kv_lo"], case["kv_hi"]) if op == "attend" else [case["tokens"]]
    blocks = max(1, _pages(lens, page))
    order = torch.randperm(blocks, generator=g, device="cuda")
    if op == "attend":
        need = torch.tensor([(n + page - 1) // page for n in lens], device="cuda")
        cols = max(1, int(need.max()))
        first = torch.cumsum(need, 0) - need
        at = (first[:, None] + torch.arange(cols, device="cuda")).clamp(max=blocks - 1)
        s["table"] = torch.where(torch.arange(cols, device="cuda") < need[:, None], order[at], 0).to(torch.int32)
        s["query"] = _normal(g, (case["batch"] * case["q_len"], kvh * case["group"], DIM), dtype, 1.3)
        s["q_lens"] = torch.full((case["batch"],), case["q_len"], dtype=torch.int64, device="cuda")
        s["kv_lens"] = torch.tensor(lens, dtype=torch.int64, device="cuda")
        s["q_len"] = case["q_len"]
    else:
        t = torch.arange(case["tokens"], device="cuda")
        s["slots"] = order[t // page] * page + t % page
    # a few of a head's key channels are several times larger than the rest
    loud = 1 + 4.0 * (torch.rand((kvh, DIM), generator=g, device="cuda") < 0.04)
    if op == "store":
        # one projection's rows: every token's keys, then its values
        s["kv"] = _normal(g, (case["tokens"], 2, kvh, DIM), dtype)
        s["kv"][:, 0] *= loud
        s["caches"] = [torch.zeros((blocks, page, kvh, ROW), dtype=torch.uint8, device="cuda") for _ in range(2)]
    else:
        s["caches"] = []
        for k in range(2):
            x = _normal(g, (blocks * page, kvh, DIM), torch.float32)
            s["caches"].append(_pack(x.mul_(loud) if k == 0 else x).view(blocks, page, kvh, ROW))
    return s


def run(s):
    return (_run_own if own else _run_plain)[s["op"]](s)


def work(case):
    e, op = BYTES[case["dtype"]], case["op"]
    if op == "logprobs":
        N, V, k = case["rows"], case["vocab"], case["top"]
        return {"bytes": N * (V * e + 8 + 4 + 4 + 8 + 12 * k), "flops": 5 * N * V}
    kvh = case["kv_heads"]
    if op == "attend":
        lens, H, q = _spread(case["batch"], case["kv_lo"], case["kv_hi"]), kvh * case["group"], case["q_len"]
        pairs = sum(max(0, n - i) for n in lens for i in range(q))
        return {"bytes": sum(lens) * kvh * 2 * ROW + case["batch"] * q * H * (2 * DIM * e + 4), "flops": 4 * pairs * H * DIM}
    rows = 2 * case["tokens"] * kvh
    return {"bytes": rows * (DIM * e + ROW) * (2 if op == "store" else 1), "flops": rows * DIM * (4 if op == "store" else 2)}


# ------------------------------------------------------------------ the framework's kernels


def _own_attend(s):
    return torch.ops.npu.cascade_quant_decode(s["query"], *s["caches"], s["table"], s["q_lens"], s["kv_lens"], s["q_len"],
                                              SCALE, True)


def _own_store(s):
    torch.ops.npu.cascade_quant_write(s["kv"][:, 0], s["kv"][:, 1], *s["caches"], s["slots"])
    return torch.ops.npu.cascade_quant_read(*s["caches"], s["slots"], s["dtype"])


def _own_read(s):
    return torch.ops.npu.cascade_quant_read(*s["caches"], s["slots"], s["dtype"])


def _own_logprobs(s):
    return torch.ops.npu.cascade_token_logprobs(s["logits"], s["tokens"], s["top"])


# ------------------------------------------------------------------ the plain forms


def _pack(x):
    """Rows [.., 128] as cache rows [.., 80]: the code of value d is nibble d % 8 of the 32-bit word
    4 ((d % 32) / 8) + d / 32; then the groups' centres and scales."""
    x = x.float().unflatten(-1, (DIM // GROUP, GROUP))
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    centre, scale = ((lo + hi) * 0.5).half(), ((hi - lo) / 15.0).half()
    by = torch.where(scale > 0, 1.0 / scale.float(), 0.0)
    code = torch.round((x - centre.float()) * by + 7.5).clamp(0, 15).to(torch.uint8)
    code = code.unflatten(-1, (4, 4, 2))                       # [.., group, eight, byte, nibble]
    code = (code[..., 0] | (code[..., 1] << 4)).transpose(-3, -2).flatten(-3)
    par = torch.cat([centre, scale], -1).flatten(-2).view(torch.uint8)
    return torch.cat([code, par], -1)


def _unpack(rows):
    """Cache rows [.., 80] as the values that they stand for [.., 128] in 32 bits."""
    code = rows[..., : DIM // 2].unflatten(-1, (4, DIM // GROUP, 4)).transpose(-3, -2)   # [.., group, eight, byte]
    code = torch.stack([code & 15, code >> 4], -1).flatten(-3).float()                   # [.., group, 32]
    par = rows[..., DIM // 2:].contiguous().view(torch.float16).unflatten(-1, (-1, 2)).float()
    return ((code - 7.5) * par[..., 1:] + par[..., :1]).flatten(-2)


def _plain_attend(s):
    B, page = s["table"].shape[0], s["caches"][0].shape[1]
    T, H, _ = s["query"].shape
    kvh, q_len = s["caches"][0].shape[2], s["q_len"]
    t = torch.arange(s["table"].shape[1] * page, device="cuda")
    k, v = (_unpack(c[s["table"].long()].flatten(1, 2).transpose(1, 2)) for c in s["caches"])   # [B, kv head, t, 128]
    q = s["query"].float().view(B, q_len, kvh, -1, DIM).permute(0, 2, 1, 3, 4).flatten(2, 3)   # [B, kv head, rows, 128]
    last = s["kv_lens"][:, None] - q_len + torch.arange(q_len, device="cuda")
    seen = (t <= last[..., None]).repeat_interleave(H // kvh, 1)[:, None]                        # [B, 1, rows, t]
    scores = torch.where(seen, torch.matmul(q, k.transpose(-1, -2)) * SCALE, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(torch.isinf(top), 0.0, top))
    total = e.sum(-1, keepdim=True)
    v = torch.where((t < s["kv_lens"][:, None])[:, None, :, None], v, 0.0)
    out = torch.matmul(e / torch.where(total > 0, total, 1.0), v)
    lse = torch.log(total) + top
    back = lambda x: x.unflatten(2, (q_len, -1)).permute(0, 2, 1, 3, 4).reshape(T, H, -1)  # noqa: E731
    return back(out).to(s["dtype"]), back(lse).reshape(T * H)


def _plain_read(s):
    return tuple(_unpack(c.flatten(0, 1)[s["slots"]]).to(s["dtype"]) for c in s["caches"])


def _plain_store(s):
    s["caches"][0].flatten(0, 1)[s["slots"]] = _pack(s["kv"][:, 0])
    s["caches"][1].flatten(0, 1)[s["slots"]] = _pack(s["kv"][:, 1])
    return _plain_read(s)


def _plain_logprobs(s):
    x, k = s["logits"].float(), s["top"]
    V = x.shape[1]
    top = x.amax(-1, keepdim=True)
    d = x - top
    e = torch.exp(d)
    total = e.sum(-1, keepdim=True)
    norm = torch.log(total)
    entropy = norm - (e * d).sum(-1, keepdim=True) / total
    tokens = s["tokens"][:, None]
    mine, at = x.gather(1, tokens), torch.arange(V, device="cuda")
    rank = ((x > mine) | ((x == mine) & (at < tokens))).sum(-1)
    # the order: larger logits first, lower indices first among equals
    bits = x.view(torch.int32).long()
    order = torch.where(bits >= 0, bits, -(bits & 0x7FFFFFFF)) * (1 << 32) + (V - 1 - at)
    best = V - 1 - (torch.topk(order, k, -1).values & 0xFFFFFFFF)
    return ((d.gather(1, tokens) - norm).squeeze(1), entropy.squeeze(1), rank, d.gather(1, best) - norm, best)


_run_own = {"attend": _own_attend, "store": _own_store, "read": _own_read, "logprobs": _own_logprobs}
_run_plain = {"attend": _plain_attend, "store": _plain_store, "read": _plain_read, "logprobs": _plain_logprobs}


# ------------------------------------------------------------------ the definitions in 64 bits


def _values(rows):
    """The values of cache rows in 64 bits, by value: byte 16 (d % 32 / 8) + 4 (d / 32) + d % 8 / 2, low nibble first."""
    d = torch.arange(DIM, device=rows.device)
    byte = rows[..., 16 * (d % 32 // 8) + 4 * (d // 32) + d % 8 // 2].int()
    code = (byte >> (4 * (d % 2)).int()) & 15
    par = rows[..., 64:].contiguous().view(torch.float16).double()
    return (code.double() - 7.5) * par[..., 2 * (d // 32) + 1] + par[..., 2 * (d // 32)]


def _nearest(x):
    """What quantising makes of x, in 64 bits but for the format's centre and scale."""
    x = x.double().unflatten(-1, (-1, GROUP))
    lo, hi = x.min(-1, keepdim=True).values, x.max(-1, keepdim=True).values
    centre, scale = ((lo + hi) / 2).half().double(), ((hi - lo) / 15).half().double()
    step = torch.where(scale > 0, ((x - centre) / torch.where(scale > 0, scale, 1.0) + 7.5).round().clamp(0, 15), 7.5)
    return ((step - 7.5) * scale + centre).flatten(-2)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "store":
        return _nearest(s["kv"][:, 0]), _nearest(s["kv"][:, 1])
    if case["op"] == "read":
        return tuple(_values(c.view(-1, *c.shape[2:])[s["slots"]]) for c in s["caches"])
    if case["op"] == "logprobs":
        parts = [], [], []
        for i in range(0, case["rows"], 256):
            p = torch.log_softmax(s["logits"][i : i + 256].double(), -1)
            parts[0].append(p.gather(1, s["tokens"][i : i + 256, None]).squeeze(1))
            parts[1].append(-(p.exp() * p).sum(-1))
            parts[2].append(p.topk(case["top"], -1).values)
        return torch.cat(parts[0]), torch.cat(parts[1]), None, torch.cat(parts[2]), None
    page, q_len, (T, H, _) = case["page"], case["q_len"], s["query"].shape
    out = torch.zeros((T, H, DIM), dtype=torch.float64, device="cuda")
    lse = torch.full((T, H), float("-inf"), dtype=torch.float64, device="cuda")
    i = torch.arange(q_len, device="cuda")[:, None]
    for b, n in enumerate(s["kv_lens"].tolist()):
        ids = s["table"][b, : (n + page - 1) // page].long()
        k, v = (_values(c[ids].view(-1, *c.shape[2:])[:n]) for c in s["caches"])
        for h in range(H):
            mine = slice(b * q_len, (b + 1) * q_len)
            scores = s["query"][mine, h].double() @ k[:, h // case["group"]].T * SCALE
            scores = scores.masked_fill(torch.arange(n, device="cuda") > n - q_len + i, float("-inf"))
            l = torch.logsumexp(scores, -1) if n else lse[mine, h]
            p = torch.exp(scores - torch.where(torch.isinf(l), 0.0, l)[:, None])
            out[mine, h], lse[mine, h] = p @ v[:, h // case["group"]], l
    return out, lse.reshape(-1)
