"""The operators of serving with a paged latent cache, as measured work: attention
over latents (absorbed for decode, expanded for prompts), the pages of the cache
(fork, free, compact) and the verification of drafted tokens.

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

LATENT, ROPE = 512, 64        # a token's cache row: 512 latent values, 64 rotary ones
NOPE, VDIM = 128, 128         # a head's expanded key (without the rotary part) and value
SCALE = (NOPE + ROPE) ** -0.5
GOLDEN = 0.6180339887498949
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
ACCEPT = 0.8                  # share of drafted tokens that prepare()'s distributions accept, roughly


def listed():
    return [
        # one user's chat on one of eight GPUs (16 of 128 heads): nothing but latency
        {"name": "decode, one request", "op": "decode", "batch": 1, "heads": 16, "q_len": 1, "kv_lo": 700, "kv_hi": 700,
         "page": 64, "dtype": "bf16"},
        # a batch of mixed chats, heads sharded, small pages
        {"name": "decode, sharded heads", "op": "decode", "batch": 48, "heads": 16, "q_len": 1, "kv_lo": 1, "kv_hi": 6001,
         "page": 16, "dtype": "bf16"},
        # data-parallel attention: every head on this GPU, a full batch of long chats
        {"name": "decode, all heads", "op": "decode", "batch": 128, "heads": 128, "q_len": 1, "kv_lo": 1500,
         "kv_hi": 8200, "page": 64, "dtype": "bf16"},
        # the target model's pass over three drafted tokens and the one before them
        {"name": "decode, drafted tokens", "op": "decode", "batch": 24, "heads": 128, "q_len": 4, "kv_lo": 4,
         "kv_hi": 5003, "page": 32, "dtype": "fp16"},
        # a handful of short prompts
        {"name": "prompt, short", "op": "prompt", "batch": 5, "heads": 16, "q_lo": 1, "q_hi": 333, "context": 0,
         "dtype": "bf16"},
        # a chunk of a long prompt behind the context that is in the cache already
        {"name": "prompt, chunk", "op": "prompt", "batch": 2, "heads": 32, "q_lo": 1000, "q_hi": 1024, "context": 4001,
         "dtype": "fp16"},
        # two long prompts at once
        {"name": "prompt, long", "op": "prompt", "batch": 2, "heads": 16, "q_lo": 6100, "q_hi": 8192, "context": 0,
         "dtype": "bf16"},
        # a few requests with three drafted tokens each
        {"name": "verify, small", "op": "verify", "batch": 4, "drafts": 3, "vocab": 32000, "dtype": "fp32"},
        # a full batch over a large vocabulary
        {"name": "verify, large", "op": "verify", "batch": 128, "drafts": 4, "vocab": 128256, "dtype": "fp32"},
        # requests that split into several samples: shared pages, a copy of the last one
        {"name": "pages, fork", "op": "fork", "rows": 64, "children": 192, "kv_lo": 1, "kv_hi": 4000, "page": 64,
         "layers": 6, "spare": 1.1, "dtype": "bf16"},
        # rejected drafts and finished requests give their pages back after a step
        {"name": "pages, free", "op": "free", "rows": 256, "kv_lo": 0, "kv_hi": 6000, "page": 64, "dtype": "bf16"},
        # the cache of a quieter hour moves to the front of its memory
        {"name": "pages, compact", "op": "compact", "rows": 48, "kv_lo": 10, "kv_hi": 4000, "page": 32, "layers": 8,
         "spare": 2.0, "dtype": "bf16"},
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(lo * (hi / lo) ** rng.random()))

    op = rng.choice(["decode", "decode", "prompt", "prompt", "verify", "fork", "free", "compact"])
    two = rng.choice(["bf16", "fp16"])
    if op == "decode":
        batch, heads, q_len = log(1, 128), rng.choice([4, 16, 20, 32, 64, 128]), rng.choice([1, 1, 1, 2, 3, 5])
        hi = log(1, 16000)
        hi = max(1, min(hi, 620000 // batch, 78000000 // (batch * heads * q_len)))
        return {"op": op, "batch": batch, "heads": heads, "q_len": q_len, "kv_lo": rng.randint(0, hi), "kv_hi": hi,
                "page": rng.choice([16, 32, 64, 128]), "dtype": two}
    if op == "prompt":
        batch, heads = log(1, 16), rng.choice([1, 4, 8, 16, 32])
        hi, context = log(1, 4000), rng.choice([0, 0, log(1, 6000)])
        hi = max(1, min(hi, int(1500000000 / (batch * heads * (hi + context)))))
        return {"op": op, "batch": batch, "heads": heads, "q_lo": rng.randint(1, hi), "q_hi": hi, "context": context,
                "dtype": two}
    if op == "verify":
        vocab = log(1000, 128256)
        return {"op": op, "batch": max(1, min(log(1, 128), 16000000 // vocab)), "drafts": rng.randint(1, 7),
                "vocab": vocab, "dtype": rng.choice(["fp32", "fp32", "bf16", "fp16"])}
    page, hi = rng.choice([16, 32, 64, 128]), log(1, 4000)
    if op == "free":
        return {"op": op, "rows": log(1, 256), "kv_lo": rng.randint(0, hi), "kv_hi": hi, "page": page, "dtype": two}
    rows = max(1, min(log(1, 64), 150000 // hi))
    case = {"op": op, "rows": rows, "kv_lo": rng.randint(0, hi), "kv_hi": hi, "page": page, "layers": rng.randint(1, 8),
            "spare": rng.choice([1.02, 1.5, 2.0]), "dtype": two}
    if op == "fork":
        case["children"] = max(1, min(log(1, 192), 16000 // page))
    return case


def _spread(n, lo, hi):
    """n whole numbers over [lo, hi], the same for every seed (work() counts them)."""
    return [lo + int((hi - lo + 1) * ((i * GOLDEN + 0.5) % 1.0)) for i in range(n)]


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * scale).to(dtype)


def _table(g, lens, page, blocks):
    """A block table over `blocks` pages in an order of its own, -1 where a row has no page."""
    need = [(n + page - 1) // page for n in lens]
    cols = max(1, max(need))
    order = torch.randperm(blocks, generator=g, device="cuda").to(torch.int32)
    have = torch.tensor(need, device="cuda")
    first = torch.cumsum(have, 0) - have
    col = torch.arange(cols, device="cuda")
    at = (first[:, None] + col).clamp(max=blocks - 1)
    return torch.where(col < have[:, None], order[at], -1).to(torch.int32).contiguous()


def _pages(lens, page):
    return sum((n + page - 1) // page for n in lens)


def prepare(case, seed):
    if own:
        here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vllm-hust-cascade-kernel_b200")
        if here not in sys.path:
            sys.path.insert(0, here)
        import cascade_kernel  # noqa: F401  registers torch.ops.npu.*
    g, op, dtype = _generator(seed), case["op"], DTYPES[case["dtype"]]
    s = {"op": op}
    if op == "decode":
        lens = _spread(case["batch"], case["kv_lo"], case["kv_hi"])
        blocks = max(1, _pages(lens, case["page"]))
        # a normalised latent has values of about one; the absorbed query's products with it are a few wide
        s["query"] = _normal(g, (case["batch"] * case["q_len"], case["heads"], LATENT + ROPE), dtype, 1.2)
        s["cache"] = _normal(g, (blocks, case["page"], LATENT + ROPE), dtype)
        s["table"] = torch.where((t := _table(g, lens, case["page"], blocks)) < 0, 0, t)
        s["q_lens"] = torch.full((case["batch"],), case["q_len"], dtype=torch.int64, device="cuda")
        s["kv_lens"] = torch.tensor(lens, dtype=torch.int64, device="cuda")
        s["q_len"] = case["q_len"]
    elif op == "prompt":
        q_lens = _spread(case["batch"], case["q_lo"], case["q_hi"])
        kv_lens = [n + case["context"] for n in q_lens]
        T, S, H = sum(q_lens), sum(kv_lens), case["heads"]
        s["query"] = _normal(g, (T, H, NOPE + ROPE), dtype, 1.5)
        s["kv"] = _normal(g, (S, H, NOPE + VDIM), dtype)  # as the up-projection writes it: a head's key, then its value
        s["k_rope"] = _normal(g, (S, ROPE), dtype)
        s["cu_q"] = torch.tensor([0] + q_lens, dtype=torch.int64).cumsum(0).cuda()
        s["cu_kv"] = torch.tensor([0] + kv_lens, dtype=torch.int64).cumsum(0).cuda()
        s["max_q"], s["max_kv"] = max(q_lens), max(kv_lens)
    elif op == "verify":
        B, K, V = case["batch"], case["drafts"], case["vocab"]
        logits = torch.randn((B, K + 1, V), generator=g, device="cuda") * 2.5
        s["target"] = torch.softmax(logits, -1).to(dtype)
        logits = logits[:, :K] + torch.randn((B, K, V), generator=g, device="cuda") * 0.5
        draft = torch.softmax(logits, -1)
        s["draft"] = draft.to(dtype)
        s["noise"] = torch.empty((B, V), device="cuda").exponential_(generator=g).clamp_(min=1e-30)
        pick = torch.empty((B, K, V), device="cuda").exponential_(generator=g).clamp_(min=1e-30)
        s["tokens"] = torch.argmax(draft / pick, -1)
        s["lens"] = torch.randint(0, K + 1, (B,), generator=g, device="cuda").clamp_(min=min(K, 2))
        s["uniform"] = torch.rand((B, K), generator=g, device="cuda")
    else:
        lens = _spread(case["rows"], case["kv_lo"], case["kv_hi"])
        used = _pages(lens, case["page"])
        blocks = max(4, int(used * case.get("spare", 1.5)) + 1)
        s["page"], s["table"] = case["page"], _table(g, lens, case["page"], blocks)
        s["kv_lens"] = torch.tensor(lens, dtype=torch.int64, device="cuda")
        flat = s["table"].reshape(-1)
        s["refs"] = torch.bincount(flat[flat >= 0].long(), minlength=blocks).to(torch.int32)
        s["pools"] = [_normal(g, (blocks, case["page"], LATENT + ROPE), dtype) for _ in range(case.get("layers", 0))]
        if op == "fork":
            s["parents"] = torch.randint(0, case["rows"], (case["children"],), generator=g, device="cuda")
        if op == "free":
            # one request in eight has ended, the others give back up to five tokens
            back = torch.randint(0, 6, (case["rows"],), generator=g, device="cuda")
            done = torch.randint(0, 8, (case["rows"],), generator=g, device="cuda") == 0
            s["keep"] = torch.where(done, 0, s["kv_lens"] - back).clamp_(min=0)
    return s


def run(s):
    return (_run_own if own else _run_plain)[s["op"]](s)


def work(case):
    e, op = BYTES[case["dtype"]], case["op"]
    if op == "decode":
        lens, rows = _spread(case["batch"], case["kv_lo"], case["kv_hi"]), case["heads"]
        T = case["batch"] * case["q_len"]
        pairs = sum(max(0, n - i) for n in lens for i in range(case["q_len"]))
        return {"bytes": sum(lens) * (LATENT + ROPE) * e + T * rows * ((2 * LATENT + ROPE) * e + 4),
                "flops": 2 * pairs * rows * (2 * LATENT + ROPE)}
    if op == "prompt":
        q, H, c = _spread(case["batch"], case["q_lo"], case["q_hi"]), case["heads"], case["context"]
        T, S = sum(q), sum(q) + c * len(q)
        pairs = sum(n * c + n * (n + 1) // 2 for n in q)
        return {"bytes": T * H * ((NOPE + ROPE + VDIM) * e + 4) + S * (H * (NOPE + VDIM) + ROPE) * e,
                "flops": 2 * pairs * H * (NOPE + ROPE + VDIM)}
    if op == "verify":
        refused = 1 - ACCEPT ** case["drafts"]
        return {"bytes": case["batch"] * case["vocab"] * (e + 4 + e * refused), "flops": 3 * case["batch"] * case["vocab"]}
    lens = _spread(case["rows"], case["kv_lo"], case["kv_hi"])
    cols, used = max(1, max((n + case["page"] - 1) // case["page"] for n in lens)), _pages(lens, case["page"])
    blocks = max(4, int(used * case.get("spare", 1.5)) + 1)
    index = 8 * blocks + 8 * case["rows"] * cols + 16 * case["rows"]
    row = (LATENT + ROPE) * e
    if op == "fork":
        tail = sum(n % case["page"] for n in lens) / len(lens)
        return {"bytes": index + 4 * case["children"] * cols + 2 * case["children"] * case["layers"] * tail * row, "flops": 0}
    if op == "compact":
        moved = used * (1 - used / blocks)
        return {"bytes": index + 2 * moved * case["layers"] * case["page"] * row, "flops": 0}
    return {"bytes": index, "flops": 0}


# ------------------------------------------------------------------ the framework's kernels


def _own_decode(s):
    return torch.ops.npu.cascade_latent_decode(s["query"], s["cache"], s["table"], s["q_lens"], s["kv_lens"], s["q_len"],
                                               SCALE, True)


def _own_prompt(s):
    k, v = s["kv"].split([NOPE, VDIM], -1)
    return torch.ops.npu.cascade_latent_prefill(s["query"], k, s["k_rope"], v, s["cu_q"], s["cu_kv"], s["max_q"], SCALE,
                                                True)


def _own_verify(s):
    return torch.ops.npu.cascade_verify_drafts(s["tokens"], s["lens"], s["draft"], s["target"], s["uniform"], s["noise"])


def _own_fork(s):
    table, lens, refs = torch.ops.npu.cascade_page_fork(s["pools"], s["table"], s["kv_lens"], s["refs"], s["parents"])
    return table, lens, refs, s["pools"]


def _own_free(s):
    return torch.ops.npu.cascade_page_free(s["table"], s["kv_lens"], s["refs"], s["keep"], s["page"])


def _own_compact(s):
    table, refs, live = torch.ops.npu.cascade_page_compact(s["pools"], s["table"], s["kv_lens"], s["refs"])
    return table, refs, live, s["pools"]


# ------------------------------------------------------------------ the plain forms


def _softmax(scores, seen):
    """exp(scores) over the last axis where `seen`, normalised, and its log sum; rows that see nothing give 0 and -inf."""
    scores = torch.where(seen, scores, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(torch.isinf(top), 0.0, top))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total > 0, total, 1.0), (torch.log(total) + top).squeeze(-1)


def _plain_decode(s):
    B, page = s["table"].shape[0], s["cache"].shape[1]
    T, H, D = s["query"].shape
    t = torch.arange(s["table"].shape[1] * page, device="cuda")
    kv = s["cache"][s["table"].long()].reshape(B, -1, D).float()
    kv = torch.where((t < s["kv_lens"][:, None])[..., None], kv, 0.0)
    scores = torch.matmul(s["query"].float().view(B, -1, D), kv.transpose(1, 2)) * SCALE
    last = s["kv_lens"][:, None] - s["q_len"] + torch.arange(s["q_len"], device="cuda")  # a token's last key
    p, lse = _softmax(scores.view(B, s["q_len"], H, -1), t <= last[:, :, None, None])
    out = torch.matmul(p.view(B, s["q_len"] * H, -1), kv[..., :LATENT])
    return out.view(T, H, LATENT).to(s["query"].dtype), lse.reshape(T * H)


def _plain_prompt(s):
    (T, H, _), B = s["query"].shape, s["cu_q"].numel() - 1
    i, t = torch.arange(s["max_q"], device="cuda"), torch.arange(s["max_kv"], device="cuda")
    n, m = s["cu_q"].diff()[:, None], s["cu_kv"].diff()[:, None]
    at_q = (s["cu_q"][:-1, None] + i).clamp(max=T - 1)
    at_kv = (s["cu_kv"][:-1, None] + t).clamp(max=s["kv"].shape[0] - 1)
    real = (t < m)[..., None, None]
    kv = torch.where(real, s["kv"][at_kv].float(), 0.0)
    rope = torch.where(real, s["k_rope"][at_kv][:, :, None].float(), 0.0).expand(-1, -1, H, -1)
    key = torch.cat([kv[..., :NOPE], rope], -1).permute(0, 2, 3, 1)
    scores = torch.matmul(s["query"][at_q].float().transpose(1, 2), key) * SCALE
    seen = (t <= (m - n)[..., None] + i[:, None]) & (t < m[..., None])
    p, lse = _softmax(scores, seen[:, None])
    out = torch.matmul(p, kv[..., NOPE:].transpose(1, 2)).transpose(1, 2)
    return out[i < n].to(s["query"].dtype), lse.transpose(1, 2)[i < n].reshape(T * H)


def _plain_verify(s):
    (B, K), n = s["tokens"].shape, s["lens"]
    row, k = torch.arange(B, device="cuda"), torch.arange(K, device="cuda")
    p = s["target"][:, :K].gather(-1, s["tokens"][..., None]).squeeze(-1).float()
    q = s["draft"].gather(-1, s["tokens"][..., None]).squeeze(-1).float()
    good = (s["uniform"] * q < p) & (k < n[:, None])
    taken = good.long().cumprod(-1).sum(-1)  # tokens before the first refusal
    p = s["target"][row, taken].float()
    q = torch.where((taken < n)[:, None], s["draft"][row, taken.clamp(max=K - 1)].float(), 0.0)
    left = (p - q).clamp(min=0.0)
    left = torch.where((left > 0).any(-1, keepdim=True), left, p)
    extra = torch.argmax(left / s["noise"], -1)
    slot = torch.arange(K + 1, device="cuda")
    kept = torch.cat([s["tokens"], s["tokens"][:, :1]], 1)
    out = torch.where(slot < taken[:, None], kept, -1)
    return torch.where(slot == taken[:, None], extra[:, None], out), taken


def _put(pool, dst, src, rows):
    new = torch.where((torch.arange(pool.shape[1], device="cuda") < rows[:, None])[..., None], pool[src], pool[dst])
    pool[dst] = new
    return pool


def _plain_fork(s):
    page, refs, parents = s["page"], s["refs"], s["parents"]
    n = s["kv_lens"][parents]
    full, tail = n // page, n % page
    free = torch.nonzero(refs == 0).squeeze(1)
    rank = torch.cumsum(tail > 0, 0) - 1
    ok = (tail == 0) | (rank < free.numel())
    mine = ok & (tail > 0)
    fresh = torch.cat([free, free.new_zeros(1)])[rank.clamp(0, free.numel())]
    col = torch.arange(s["table"].shape[1], device="cuda")
    old = s["table"][parents]
    shared = (col < full[:, None]) & ok[:, None]
    table = torch.where(shared, old, -1)
    table = torch.where((col == full[:, None]) & mine[:, None], fresh[:, None].int(), table)
    refs = refs + torch.bincount(table[table >= 0].long(), minlength=refs.numel()).int()
    src = old.gather(1, full.clamp(max=old.shape[1] - 1)[:, None]).squeeze(1).long()
    pools = [_put(pool, fresh[mine], src[mine], tail[mine]) for pool in s["pools"]]
    return table, torch.where(ok, n, -1), refs, pools


def _plain_free(s):
    page, n = s["page"], s["kv_lens"]
    keep = torch.minimum(s["keep"].clamp(min=0), n)
    col = torch.arange(s["table"].shape[1], device="cuda")
    have, hold = (n + page - 1) // page, (keep + page - 1) // page
    gone = (col >= hold[:, None]) & (col < have[:, None])
    refs = s["refs"] - torch.bincount(s["table"][gone].long(), minlength=s["refs"].numel()).int()
    return torch.where(col < hold[:, None], s["table"], -1), keep, refs


def _plain_compact(s):
    refs, table = s["refs"], s["table"]
    live, ids = refs > 0, torch.arange(refs.numel(), device="cuda")
    count = live.sum(dtype=torch.int32)
    src, dst = torch.nonzero(live & (ids >= count)).squeeze(1), torch.nonzero(~live & (ids < count)).squeeze(1)
    to = ids.clone()
    to[src] = dst
    full = torch.full_like(src, s["page"])
    pools = [_put(pool, dst, src, full) for pool in s["pools"]]
    have = (s["kv_lens"] + s["page"] - 1) // s["page"]
    col = torch.arange(table.shape[1], device="cuda")
    moved = torch.where(col < have[:, None], to[table.clamp(min=0).long()].int(), -1)
    new = torch.zeros_like(refs).scatter_add_(0, to, torch.where(live, refs, 0))
    return moved, new, count.reshape(1), pools


_run_own = {"decode": _own_decode, "prompt": _own_prompt, "verify": _own_verify, "fork": _own_fork, "free": _own_free,
            "compact": _own_compact}
_run_plain = {"decode": _plain_decode, "prompt": _plain_prompt, "verify": _plain_verify, "fork": _plain_fork,
              "free": _plain_free, "compact": _plain_compact}


# ------------------------------------------------------------------ the definitions in 64 bits


def _attend(q, k, v, n, first):
    """One head group: q [.., i, d] over k, v [.., t, d]; query i sees keys 0 .. first + i."""
    scores = torch.matmul(q, k.transpose(-1, -2)) * SCALE
    i, t = torch.arange(q.shape[-2], device="cuda")[:, None], torch.arange(n, device="cuda")
    scores = scores.masked_fill(t > first + i, float("-inf"))
    lse = torch.logsumexp(scores, -1) if n else torch.full(scores.shape[:-1], float("-inf"), device="cuda").double()
    p = torch.exp(scores - torch.where(torch.isinf(lse), 0.0, lse)[..., None])
    return torch.matmul(p, v), lse


def exact(case, seed):
    if case["op"] not in ("decode", "prompt", "verify"):
        return None
    s = prepare(case, seed)
    outs, lses = [], []
    if case["op"] == "verify":
        return None  # whole numbers: equal or not
    if case["op"] == "decode":
        page, q = case["page"], s["query"].double()
        for b, n in enumerate(s["kv_lens"].tolist()):
            ids = s["table"][b, : (n + page - 1) // page].long()
            kv = s["cache"][ids].reshape(-1, LATENT + ROPE)[:n].double()
            mine = q[b * s["q_len"] : (b + 1) * s["q_len"]].transpose(0, 1)
            o, l = _attend(mine, kv, kv[:, :LATENT], n, n - s["q_len"])
            outs.append(o.transpose(0, 1))
            lses.append(l.transpose(0, 1).reshape(-1))
        return torch.cat(outs), torch.cat(lses)
    cu_q, cu_kv = s["cu_q"].tolist(), s["cu_kv"].tolist()
    T, H, _ = s["query"].shape
    out, lse = torch.empty((T, H, VDIM), dtype=torch.float64, device="cuda"), torch.empty((T, H), dtype=torch.float64, device="cuda")
    for b in range(len(cu_q) - 1):
        q, kv = s["query"][cu_q[b] : cu_q[b + 1]], s["kv"][cu_kv[b] : cu_kv[b + 1]]
        rope = s["k_rope"][cu_kv[b] : cu_kv[b + 1]].double()
        for h in range(H):
            k = torch.cat([kv[:, h, :NOPE].double(), rope], 1)
            o, l = _attend(q[:, h].double(), k, kv[:, h, NOPE:].double(), k.shape[0], k.shape[0] - q.shape[0])
            out[cu_q[b] : cu_q[b + 1], h], lse[cu_q[b] : cu_q[b + 1], h] = o, l
    return out, lse.reshape(-1)
