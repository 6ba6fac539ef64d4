"""Speculative decoding over a paged latent cache, one attention layer of a random model.

    python examples/latent_speculative.py [--samples 8] [--prompt 700] [--steps 4] [--drafts 3]

A prompt is attended in the expanded form (every head's keys and values are
projected up from the latents) while its latents go to the cache; the sequence
forks into samples that share its pages; each step, drafted tokens are appended
and attended in the absorbed form, verified against the target's
probabilities, and the rejected ones' pages are given back. At the end half the
samples leave and the cache is compacted.
"""
import argparse
import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "vllm-hust-cascade-kernel_b200"))

import torch  # noqa: E402

import cascade_kernel  # noqa: E402,F401  registers torch.ops.npu.*
from cascade_kernel.latent import LATENT, ROPE, LatentCache  # noqa: E402

NOPE, VDIM = 128, 128
SCALE = (NOPE + ROPE) ** -0.5


class Layer:
    """Random projections of one latent attention layer and a vocabulary; positions carry no rotation here."""

    def __init__(self, heads, hidden, vocab, g):
        def w(*shape, fan):
            return (torch.randn(shape, generator=g, device="cuda") * fan ** -0.5).to(torch.bfloat16)

        self.embed = w(vocab, hidden, fan=1)
        self.to_latent = w(hidden, LATENT + ROPE, fan=hidden)
        self.to_query = w(hidden, heads * (NOPE + ROPE), fan=hidden)
        self.up_key, self.up_value = w(heads, NOPE, LATENT, fan=LATENT), w(heads, VDIM, LATENT, fan=LATENT)
        self.out, self.head = w(heads * VDIM, hidden, fan=heads * VDIM), w(hidden, vocab, fan=hidden)
        self.heads = heads

    def latents(self, tokens):
        return self.embed[tokens] @ self.to_latent

    def query(self, tokens):
        return (self.embed[tokens] @ self.to_query).view(-1, self.heads, NOPE + ROPE)

    def absorbed_query(self, tokens):
        q = self.query(tokens)
        return torch.cat([torch.einsum("thd,hdc->thc", q[..., :NOPE], self.up_key), q[..., NOPE:]], -1)

    def expand(self, latents):
        c = latents[:, :LATENT]
        return torch.einsum("tc,hdc->thd", c, self.up_key), torch.einsum("tc,hdc->thd", c, self.up_value)

    def probs(self, tokens, values):
        hidden = self.embed[tokens] + values.reshape(values.shape[0], -1) @ self.out
        return torch.softmax((hidden @ self.head).float(), -1)


def run(samples=8, prompt=700, steps=4, drafts=3, heads=16, hidden=512, vocab=2000, page=64, seed=0, log=print):
    g = torch.Generator(device="cuda").manual_seed(seed)
    npu = torch.ops.npu
    layer = Layer(heads, hidden, vocab, g)
    longest = prompt + steps * (drafts + 1) + 1
    cols = -(-longest // page)
    cache = LatentCache(1, cols * (samples + 1) + 8, page, 1, cols)

    # the prompt, expanded, and its latents into the cache
    tokens = torch.randint(0, vocab, (prompt,), generator=g, device="cuda")
    latents = layer.latents(tokens)
    cache.grow(torch.tensor([prompt], device="cuda"))
    cache.write(0, latents, [prompt])
    key, value = layer.expand(latents)
    cu = torch.tensor([0, prompt], dtype=torch.int64, device="cuda")
    attended, _ = npu.cascade_latent_prefill(layer.query(tokens), key, latents[:, LATENT:].contiguous(), value, cu, cu,
                                             prompt, SCALE, True)
    p = layer.probs(tokens[-1:], attended[-1:])

    # the last prompt token once more in the absorbed form: both forms say the same
    again, _ = cache.attend(0, layer.absorbed_query(tokens[-1:]), 1, SCALE)
    again = torch.einsum("thc,hdc->thd", again, layer.up_value)
    gap = float((again.float() - attended[-1:].float()).abs().max() / attended[-1].float().abs().max())

    # the samples: rows that share the prompt's pages
    cache.fork(torch.zeros(samples, dtype=torch.int64, device="cuda"))
    last = torch.multinomial(p, samples, replacement=True, generator=g).view(samples)
    produced, accepted = [last[:, None]], 0
    for _ in range(steps):
        # a cheap draft: the model without attention
        chain, q = [last], []
        for _ in range(drafts):
            q.append(layer.probs(chain[-1], torch.zeros((samples, heads, VDIM), dtype=torch.bfloat16, device="cuda")))
            chain.append(torch.multinomial(q[-1], 1, generator=g).view(samples))
        fed = torch.stack(chain, 1)  # the last token and its drafts: all go to the cache
        before = cache.lens
        n = drafts + 1
        cache.grow(torch.full_like(before, n))
        cache.write(0, layer.latents(fed.reshape(-1)), [n] * samples)
        o, _ = cache.attend(0, layer.absorbed_query(fed.reshape(-1)), n, SCALE)
        target = layer.probs(fed.reshape(-1), torch.einsum("thc,hdc->thd", o, layer.up_value)).view(samples, n, vocab)
        out, taken = npu.cascade_verify_drafts(
            fed[:, 1:].contiguous(), torch.full((samples,), drafts, dtype=torch.int64, device="cuda"),
            torch.stack(q, 1).contiguous(), target.contiguous(), torch.rand((samples, drafts), generator=g, device="cuda"),
            torch.empty((samples, vocab), device="cuda").exponential_(generator=g))
        # the rejected drafts leave the cache; the token after the accepted ones comes next
        cache.truncate(before + 1 + taken)
        last = out.gather(1, taken[:, None]).squeeze(1)
        produced.append(out)
        accepted += int(taken.sum())
    live_before = int((cache.refs > 0).sum())
    keep = torch.where(torch.arange(samples, device="cuda") % 2 == 0, cache.lens, 0)
    cache.truncate(keep)
    live = int(cache.compact())
    log(f"prompt of {prompt} tokens: expanded and absorbed attention differ by {gap:.1e} of the largest value")
    log(f"{samples} samples x {steps} steps: {accepted} of {samples * steps * drafts} drafts accepted; pages in use "
        f"{live_before}, after half the samples left and compaction {live}")
    return {"gap": gap, "accepted": accepted, "live": live, "cache": cache, "produced": produced, "keep": keep}


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    for name, default in (("samples", 8), ("prompt", 700), ("steps", 4), ("drafts", 3)):
        ap.add_argument("--" + name, type=int, default=default)
    run(**vars(ap.parse_args()))
