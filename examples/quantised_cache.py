"""Serving from a key-value cache held in 4 bits, one attention layer of a random model.

    python examples/quantised_cache.py [--samples 8] [--prompt 900] [--chunk 256] [--steps 4]

A prompt enters the cache in chunks, quantised as it is written, and each chunk
attends to the cache as it lies. The prompt's log probabilities, against those
of attention over the unrounded keys and values, say what the 4 bits cost. The
sequence then forks into samples that share the prompt's pages; each step reads
the shared pages once for all of them, and the step's tokens come with their log
probabilities and best alternatives. At the end half the samples leave, the
cache is compacted, and the rest of a row is read back into 16 bits.
"""
import argparse
import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "vllm-hust-cascade-kernel_b200"))

import torch  # noqa: E402

import cascade_kernel  # noqa: E402,F401  registers torch.ops.npu.*
from cascade_kernel.quant import DIM, QuantCache  # noqa: E402

SCALE = DIM ** -0.5


class Layer:
    """Random projections of one layer with grouped query heads and a vocabulary; positions carry no rotation here."""

    def __init__(self, heads, kv_heads, hidden, vocab, g):
        def w(*shape, fan):
            return (torch.randn(shape, generator=g, device="cuda") * fan ** -0.5).to(torch.bfloat16)

        self.embed = w(vocab, hidden, fan=1)
        self.qkv = w(hidden, (heads + 2 * kv_heads) * DIM, fan=hidden)
        self.out, self.head = w(heads * DIM, hidden, fan=heads * DIM), w(hidden, vocab, fan=hidden)
        self.heads, self.kv_heads = heads, kv_heads

    def project(self, tokens):
        """Queries, keys and values: views of one projection's rows."""
        x = (self.embed[tokens] @ self.qkv).view(-1, self.heads + 2 * self.kv_heads, DIM)
        q, k, v = x.split([self.heads, self.kv_heads, self.kv_heads], 1)
        return q.contiguous(), k, v

    def logits(self, tokens, values):
        return (self.embed[tokens] + values.reshape(values.shape[0], -1) @ self.out) @ self.head


def plain_attention(q, k, v):
    """Causal attention over the unrounded keys and values, in 32 bits."""
    n, group = q.shape[0], q.shape[1] // k.shape[1]
    k, v = (x.float().repeat_interleave(group, 1) for x in (k, v))
    s = torch.einsum("ihd,thd->hit", q.float(), k) * SCALE
    s = s.masked_fill(torch.ones((n, n), dtype=torch.bool, device=q.device).triu(1), float("-inf"))
    return torch.einsum("hit,thd->ihd", torch.softmax(s, -1), v).to(q.dtype)


def run(samples=8, prompt=900, chunk=256, steps=4, heads=16, kv_heads=4, hidden=512, vocab=2000, page=64, seed=0, log=print):
    g = torch.Generator(device="cuda").manual_seed(seed)
    npu = torch.ops.npu
    layer = Layer(heads, kv_heads, hidden, vocab, g)
    cols = -(-(prompt + steps + 1) // page)
    cache = QuantCache(1, cols * (samples + 1) + 8, page, 1, cols, kv_heads)

    # the prompt, chunk by chunk
    tokens = torch.randint(0, vocab, (prompt,), generator=g, device="cuda")
    q, k, v = layer.project(tokens)
    parts = []
    for at in range(0, prompt, chunk):
        n = min(chunk, prompt - at)
        cache.grow(torch.tensor([n], device="cuda"))
        cache.write(0, k[at : at + n], v[at : at + n], [n])
        parts.append(cache.attend(0, q[at : at + n].contiguous(), n, SCALE)[0])
    ours = layer.logits(tokens, torch.cat(parts))
    theirs = layer.logits(tokens, plain_attention(q, k, v))
    following = torch.cat([tokens[1:], tokens[:1]])
    scored = [npu.cascade_token_logprobs(x, following, 3) for x in (ours, theirs)]
    drift = float((scored[0][0] - scored[1][0])[:-1].abs().mean())
    entropy = float(scored[1][1].mean())

    # the samples: rows that share the prompt's pages; a prefix of whole pages is read once for all
    shared = prompt // page * page
    prefix = cache.table[:, : shared // page].contiguous()
    prefix_lens = torch.tensor([shared], dtype=torch.int64, device="cuda")
    cache.fork(torch.zeros(samples, dtype=torch.int64, device="cuda"))
    noise = torch.empty((samples, vocab), device="cuda")
    pick = lambda x: (torch.log_softmax(x.float(), -1) - noise.exponential_(generator=g).log()).argmax(-1)  # noqa: E731
    last = pick(ours[-1:].expand(samples, -1))
    answers = []
    for _ in range(steps):
        q, k, v = layer.project(last)
        cache.grow(torch.ones_like(cache.lens))
        cache.write(0, k, v, [1] * samples)
        o = cache.attend_shared(0, q, prefix, prefix_lens, SCALE, shared)
        logits = layer.logits(last, o)
        last = pick(logits)
        answers.append((last, *npu.cascade_token_logprobs(logits, last, 5)))
    alone, _ = cache.attend(0, q, 1, SCALE)
    gap = float((alone.float() - o.float()).abs().max() / alone.float().abs().max())

    cache.truncate(torch.where(torch.arange(samples, device="cuda") % 2 == 0, cache.lens, 0))
    live = int(cache.compact())
    kept = [steps if i % 2 == 0 else 0 for i in range(samples)]
    back, _ = cache.read(0, kept)  # the samples' own keys
    log(f"prompt of {prompt} tokens: log probabilities {drift:.1e} off those over unrounded keys and values, on average "
        f"(entropy {entropy:.2f})")
    log(f"{samples} samples x {steps} steps: shared and own attention differ by {gap:.1e} of the largest value; mean log "
        f"probability {float(torch.stack([a[1] for a in answers]).mean()):.2f}; {live} pages in use after half of them left")
    return {"drift": drift, "entropy": entropy, "gap": gap, "answers": answers, "cache": cache, "live": live, "back": back,
            "keys": k, "scored": scored}


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    for name, default in (("samples", 8), ("prompt", 900), ("chunk", 256), ("steps", 4)):
        ap.add_argument("--" + name, type=int, default=default)
    run(**vars(ap.parse_args()))
